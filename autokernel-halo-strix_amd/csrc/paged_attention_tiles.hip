// Attention over a paged cache on the matrix cores, for gfx950.
//
// Work. The query heads that share a key head go together: a tile is the rows
// (token, head of the group) of up to R = 32 (a wave) or 32 x waves rows, token by
// token, and its keys are cut into units of a fixed number of keys. All tiles' units
// stand in one line, sequence by sequence, key head by key head, and every worker
// (a wave, or a workgroup) takes the same number of them, whatever the lengths: a
// worker that has a tile's units whole writes its rows, the others leave (maximum, sum,
// sums of products) in fp32, which a second kernel joins in the order of the workers.
//
// A unit. S^T = K Q^T puts the keys of a query into one lane pair's registers: the
// running maximum and sum are in-lane work, and the sums of products O^T = V^T P^T
// keep a query in the same lane, so rescaling them takes one factor a lane. P^T's
// registers are the product's operand as they are (16 bit: rounded once, its keys
// numbered so that both products agree); V is read from LDS transposed.
#include <algorithm>

#include "mfma_ring.h"
#include "paged_attention.h"

namespace ak {
namespace {

constexpr int kRows = 32;          // rows of a wave
constexpr int kPlanBatch = 1024;   // sequences that a workgroup lines up by itself

typedef float f32x4_v __attribute__((ext_vector_type(4)));
typedef const int32_t __attribute__((address_space(4)))* ConstI32;

// What the joining kernel does for a worker: the rows of its last tile, whose first part
// is the worker's own.
struct Job {
  int64_t token, first;  // the tile's first token of the call; its part's slot
  int head, rows, parts, pad;  // its first query head; rows 0: nothing
};

struct TileArgs {
  AttendArgs a;
  int group, per_tile;             // heads of a group, tokens of a tile
  uint32_t page_magic;             // floor(2^32 / page_size), at most 2^32 - 1
  int unit, rows;                  // keys of a unit, rows of a tile
  int workers, min_units;
  int64_t* line;                   // [batch + 1]: the units before each sequence
  Job* jobs;                       // [workers]
  float* part;                     // [2 workers][rows][DB + 2]: sums of products, maximum, sum
  float c, cap_in, cap_out;        // scores in base 2: s c, or cap_out tanh(s cap_in)
};

// Where a key lives.
__device__ __forceinline__ void key_place(const TileArgs& g, uint32_t key, uint32_t& page, uint32_t& slot) {
  const uint32_t d = (uint32_t)g.a.page_size;
  page = __umulhi(key, g.page_magic);  // the quotient or one less
  slot = key - page * d;
  if (slot >= d) {
    slot -= d;
    ++page;
  }
}

// A sequence's part in the line.
struct Seq {
  int64_t first;      // its first new token
  int count, length;  // new tokens, positions that can have keys
  int pos0;           // position of the first new token
};

__device__ __forceinline__ Seq seq_at(const TileArgs& g, int64_t b) {
  Seq s;
  int64_t count;
  sequence_tokens(g.a.seq, b, s.first, count);
  const int length = g.a.seq.lengths[b];
  s.count = (int)count;
  // (far below 0 all the same once it is: no key)
  s.pos0 = (int)max((int64_t)length - count, (int64_t)INT32_MIN / 2);
  s.length = (int)min((int64_t)length, g.a.max_pages * g.a.page_size);
  return s;
}

// The keys [lo, hi) that some token of tile t sees, in units [u0, u1) (one at least).
struct Span {
  int lo, hi, u0, u1;
};

__device__ __forceinline__ Span span_of(const TileArgs& g, const Seq& s, int t) {
  const int t0 = t * g.per_tile, t1 = min(t0 + g.per_tile, s.count);
  Span r;
  r.hi = max(min(s.pos0 + t1, s.length), 0);
  r.lo = 0;
  if (g.a.window > 0) r.lo = (int)min(max((int64_t)s.pos0 + t0 + 1 - g.a.window, (int64_t)0), (int64_t)r.hi);
  r.u0 = (uint32_t)r.lo / (uint32_t)g.unit;
  r.u1 = max((int)(((uint32_t)r.hi + g.unit - 1) / (uint32_t)g.unit), r.u0 + 1);
  return r;
}

__device__ __forceinline__ int tiles_of(const TileArgs& g, const Seq& s) { return (s.count + g.per_tile - 1) / g.per_tile; }

// Workers that a line of `total` units keeps busy; worker w has [begin(w), begin(w + 1)).
__device__ __forceinline__ int64_t active_workers(const TileArgs& g, int64_t total) {
  return max(min((int64_t)g.workers, total / g.min_units), (int64_t)1);
}
__device__ __forceinline__ int64_t begin_of(int64_t w, int64_t total, int64_t n) { return w * total / n; }
__device__ __forceinline__ int64_t worker_of(int64_t u, int64_t total, int64_t n) { return ((u + 1) * n - 1) / total; }

__device__ __forceinline__ int64_t wave_sum64(int64_t v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

// The tile of a line's unit.
struct Place {
  int64_t b;
  int h, t;        // key head, tile of the sequence
  int64_t begin;   // the tile's first unit in the line
  Seq s;
  Span k;
};

// Which head and tile of sequence b unit u is in; the sequence's units begin at `at`.
// All lanes of a wave together.
__device__ __forceinline__ void place_in_sequence(const TileArgs& g, Place& p, int64_t u, int64_t at, int64_t units) {
  const int lane = threadIdx.x & 63;
  p.s = seq_at(g, p.b);
  const int64_t each = units / g.a.kv_heads;
  int64_t rest = u - at;
  p.h = (int)(rest / each);
  rest -= (int64_t)p.h * each;
  const int n = tiles_of(g, p.s);
  int t = 0;
  if (n > 1) {
    for (;; t += 64) {
      int64_t mine = 0;
      if (t + lane < n) {
        const Span k = span_of(g, p.s, t + lane);
        mine = k.u1 - k.u0;
      }
      int64_t upto = mine;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int64_t o = __shfl_up(upto, d);
        if (lane >= d) upto += o;
      }
      const int64_t all = __shfl(upto, 63);
      if (rest < all || t + 64 >= n) {
        const uint64_t over = __ballot(upto > rest);
        const int i = over ? __builtin_ctzll(over) : 0;
        rest -= __shfl(upto - mine, i);
        t += i;
        break;
      }
      rest -= all;
    }
  }
  p.t = __builtin_amdgcn_readfirstlane(t);
  p.h = __builtin_amdgcn_readfirstlane(p.h);
  p.begin = u - rest;
  p.k = span_of(g, p.s, p.t);
}

// The sequence of unit u from the line in memory: 64 entries at a time.
__device__ __forceinline__ int64_t sequence_at(const int64_t* line, int64_t batch, int64_t u) {
  const int lane = threadIdx.x & 63;
  int64_t lo = 0, n = batch;
  while (n > 1) {
    const int64_t step = (n + 63) / 64;
    const bool le = lane * step < n && line[lo + lane * step] <= u;
    const int last = 63 - __builtin_clzll(__ballot(le) | 1);
    const int64_t next = lo + last * step;
    n = min(step, lo + n - next);
    lo = next;
  }
  // (sequences without units begin where the next one does: the last of them is ours)
  return lo;
}

__device__ __forceinline__ int64_t units_of(const TileArgs& g, const Seq& s, int first_tile, int step) {
  int64_t sum = 0;
  const int n = tiles_of(g, s);
  for (int t = first_tile; t < n; t += step) {
    const Span k = span_of(g, s, t);
    sum += k.u1 - k.u0;
  }
  return sum;
}

// Lines up the units of all sequences: a wave each, then their sums.
__global__ void __launch_bounds__(1024) attend_line_kernel(TileArgs g) {
  __shared__ int64_t sums[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t batch = g.a.seq.batch;
  for (int64_t b = wave; b < batch; b += 16) {
    const int64_t n = wave_sum64(units_of(g, seq_at(g, b), lane, 64));
    if (lane == 0) g.line[b + 1] = n * g.a.kv_heads;
  }
  if (threadIdx.x == 0) g.line[0] = 0;
  __syncthreads();
  int64_t before = 0;
  for (int64_t b0 = 0; b0 < batch; b0 += 1024) {
    const int64_t b = b0 + threadIdx.x;
    int64_t upto = b < batch ? g.line[b + 1] : 0;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t o = __shfl_up(upto, d);
      if (lane >= d) upto += o;
    }
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    int64_t add = before;
    for (int w = 0; w < 16; ++w) {
      if (w < wave) add += sums[w];
      before += sums[w];
    }
    if (b < batch) g.line[b + 1] = upto + add;
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// A unit's arithmetic
// ---------------------------------------------------------------------------
template <typename T, int DB>
struct Shape {
  static constexpr int VE = Vec16<T>::VE;
  static constexpr int kChunks = DB / VE;            // 16-byte chunks of a row
  // Rows in LDS are a chunk (K: a column of chunks is read) or two (V: two chunks of four
  // rows are read together) longer than their values, which spreads them over the banks.
  static constexpr int kRowBytes = DB * (int)sizeof(T);
  static constexpr int kPitch = kRowBytes + 16, vPitch = kRowBytes + 32;
  static constexpr int kPerLoad = 64 / kChunks;      // rows of one load of a wave
  static constexpr int kSteps = DB / (2 * VE);       // operand steps of a score
  static constexpr int kBlocks = DB / 32;            // blocks of 32 values
  static_assert(kChunks <= 64, "a row is at most one load of a wave");
};

// One operand step of S^T: 16 bytes of each operand.
__device__ __forceinline__ f32x16_t mfma_step(bf16 t, u32x4 k, u32x4 q, f32x16_t c) { return mfma32(t, k, q, c); }
__device__ __forceinline__ f32x16_t mfma_step(f16 t, u32x4 k, u32x4 q, f32x16_t c) { return mfma32(t, k, q, c); }
__device__ __forceinline__ f32x16_t mfma_step(float, u32x4 k, u32x4 q, f32x16_t c) {
  const f32x4_v a = __builtin_bit_cast(f32x4_v, k), b = __builtin_bit_cast(f32x4_v, q);
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
  return c;
}

typedef short i16x4_v __attribute__((ext_vector_type(4)));
typedef i16x4_v __attribute__((address_space(3)))* LdsI16x4;

// 4 rows x 16 columns of 16-bit values a lane group of 16, transposed.
__device__ __forceinline__ u32x2 lds_tr(const char* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsI16x4)(p)));
}

// Where a value is not finite.
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t x) {
  if constexpr (sizeof(T) == 4) return ((x & 0x7F800000u) + 0x00800000u) & 0x80000000u;
  else if constexpr (std::is_same<T, f16>::value) return ((x & 0x7C007C00u) + 0x04000400u) & 0x80008000u;
  else return ((x & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
}
// x with 0 in place of what is not finite, given not_finite(x).
template <typename T>
__device__ __forceinline__ uint32_t finite_only(uint32_t x, uint32_t bad) {
  if constexpr (sizeof(T) == 4) return bad ? 0u : x;
  else return x & ~((bad >> 15) * 0xFFFFu);
}

// The other half's value of the same query.
__device__ __forceinline__ float other_half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float both_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// A wave's rows: 32 queries, lane l and l + 32 the same one.
template <typename T, int DB>
struct Rows {
  u32x4 q[Shape<T, DB>::kSteps];
  f32x16_t o[Shape<T, DB>::kBlocks];
  float m, l;     // the running maximum (base 2; the lane's query) and this half's sum
  int lo, hi;     // the keys that the query sees
  int top, low;   // of the wave's rows: the least hi, the largest lo
  bool live;
};

// Loads the queries of rows [row0, row0 + 32) of a tile and starts their sums.
template <typename T, int DB>
__device__ __forceinline__ void rows_begin(const TileArgs& g, const Place& p, int row0, Rows<T, DB>& r) {
  using S = Shape<T, DB>;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int t0 = p.t * g.per_tile, tokens = min(g.per_tile, p.s.count - t0);
  const int row = row0 + (lane & 31);
  const int i = (uint32_t)row / (uint32_t)g.group;  // token of the tile
  r.live = i < tokens && row < g.rows;
  const int tok = min(i, tokens - 1);
  const int pos = p.s.pos0 + t0 + tok;
  r.hi = r.live ? max(min(pos + 1, p.s.length), 0) : 0;
  r.lo = g.a.window > 0 ? (int)max((int64_t)pos + 1 - g.a.window, (int64_t)0) : 0;
  // (rows past the tile's see what its last token does: nothing of theirs is kept, and they mask nothing)
  const int last = min((int)((uint32_t)(row0 + 31) / (uint32_t)g.group), tokens - 1), fst = min((int)((uint32_t)row0 / (uint32_t)g.group), tokens - 1);
  r.top = __builtin_amdgcn_readfirstlane(max(min(p.s.pos0 + t0 + fst + 1, p.s.length), 0));
  r.low = g.a.window > 0 ? __builtin_amdgcn_readfirstlane((int)max((int64_t)p.s.pos0 + t0 + last + 1 - g.a.window, (int64_t)0)) : 0;
  const T* q = static_cast<const T*>(g.a.q) + (p.s.first + t0 + tok) * g.a.q_st +
               (int64_t)(p.h * g.group + (row - i * g.group)) * g.a.q_sh;
#pragma unroll
  for (int k = 0; k < S::kSteps; ++k) {
    r.q[k] = u32x4{0, 0, 0, 0};
    const int d = (2 * k + half) * S::VE;
    if (r.live && d < g.a.dim) r.q[k] = *reinterpret_cast<const u32x4*>(q + d);
  }
#pragma unroll
  for (int b = 0; b < S::kBlocks; ++b) r.o[b] = f32x16_t{};
  r.m = kNegInf;
  r.l = 0.0f;
}

// 32 keys from `key0` on, their K and V at kl and vl in LDS (rows row0 .. row0 + 31
// there). edge: some row does not see all of them; seen: their bits that exist.
template <typename T, int DB>
__device__ __forceinline__ f32x16_t scores32(const TileArgs& g, const Rows<T, DB>& r, const char* kl, int row0) {
  using S = Shape<T, DB>;
  const int lane = threadIdx.x & 63, half = lane >> 5, row = row0 + (lane & 31);
  const char* base = kl + row * S::kPitch + 16 * half;
  f32x16_t s{};
#pragma unroll
  for (int k = 0; k < S::kSteps; ++k) s = mfma_step(T(), *reinterpret_cast<const u32x4*>(base + 32 * k), r.q[k], s);
  if (g.cap_out > 0.0f) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = g.cap_out * tanh_f32(s[i] * g.cap_in);
  }
  return s;
}

template <typename T, int DB>
__device__ __forceinline__ void hide32(const Rows<T, DB>& r, f32x16_t& s, int key0, uint32_t seen) {
  const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int j = 8 * (i / 4) + 4 * half + i % 4, key = key0 + j;
    if (key >= r.hi || key < r.lo || !((seen >> j) & 1)) s[i] = kNegInf;
  }
}

// The running maximum over N x 32 new scores, and everything so far brought to it.
template <typename T, int DB, int N>
__device__ __forceinline__ void new_maximum(const TileArgs& g, Rows<T, DB>& r, const f32x16_t (&s)[N]) {
  float top = s[0][0];
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, s[n][i]);
  top = other_half_max(top);
  const float scaled = g.cap_out > 0.0f ? top : top * g.c;
  if (__any(scaled > r.m)) {
    const float m = fmaxf(r.m, scaled);
    const float keep = r.m == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(r.m - m);
    r.m = m;
    r.l *= keep;
#pragma unroll
    for (int b = 0; b < Shape<T, DB>::kBlocks; ++b) r.o[b] *= keep;
  }
}

// The weights of 32 keys: s becomes p, the sum grows.
template <typename T, int DB>
__device__ __forceinline__ void weights32(const TileArgs& g, Rows<T, DB>& r, f32x16_t& s) {
  const float c = g.cap_out > 0.0f ? 1.0f : g.c;
  // (nothing seen yet: every score is -inf or NaN, and the weight 0 or NaN)
  const float m = r.m == kNegInf ? 0.0f : r.m;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, -m));
    r.l += s[i];
  }
}

// O^T += V^T P^T of 32 keys.
template <typename T, int DB>
__device__ __forceinline__ void values32(Rows<T, DB>& r, const f32x16_t& p, const char* vl, int row0) {
  using S = Shape<T, DB>;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  if constexpr (sizeof(T) == 2) {
    // lane group q of 16 reads rows 4 (q / 2) + 0 .. 3 and 8 further on, columns 16 (q % 2) on
    const int j = lane & 15;
    const char* base = vl + (row0 + 4 * half + (j >> 2)) * S::vPitch + 32 * ((lane >> 4) & 1) + 8 * (j & 3);
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      u32x4 b;
#pragma unroll
      for (int i = 0; i < 4; ++i) b[i] = pack2<T>(p[8 * kb + 2 * i], p[8 * kb + 2 * i + 1]);
#pragma unroll
      for (int blk = 0; blk < S::kBlocks; ++blk) {
        const u32x2 x = lds_tr(base + 16 * kb * S::vPitch + 64 * blk);
        const u32x2 y = lds_tr(base + (16 * kb + 8) * S::vPitch + 64 * blk);
        r.o[blk] = mfma32(T(), u32x4{x[0], x[1], y[0], y[1]}, b, r.o[blk]);
      }
    }
  } else {
    const char* base = vl + (row0 + 4 * half) * S::vPitch + 4 * (lane & 31);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
#pragma unroll
      for (int blk = 0; blk < S::kBlocks; ++blk) {
        const float v = *reinterpret_cast<const float*>(base + (8 * (i / 4) + i % 4) * S::vPitch + 128 * blk);
        r.o[blk] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, p[i], r.o[blk], 0, 0, 0);
      }
    }
  }
}

// What values that are not finite (left out of LDS where only some rows see them) do to
// the rows that see their keys.
template <typename T, int DB>
__device__ __forceinline__ void add_not_finite(const TileArgs& g, const Place& p, Rows<T, DB>& r, int key0, uint32_t seen) {
  const int half = (threadIdx.x & 63) >> 5;
  const T* v0 = static_cast<const T*>(g.a.v) + (int64_t)p.h * g.a.vh;
  for (int j = 0; j < 32; ++j) {
    if (!((seen >> j) & 1)) continue;
    const int key = key0 + j;
    uint32_t i, slot;
    key_place(g, (uint32_t)key, i, slot);
    const int64_t page = g.a.pages[p.b * g.a.ld_pages + i];  // (there: its bit is set)
    const T* v = v0 + page * g.a.vp + (int64_t)slot * g.a.vs;
    const bool sees = key < r.hi && key >= r.lo;
#pragma unroll
    for (int blk = 0; blk < Shape<T, DB>::kBlocks; ++blk)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int d = 32 * blk + 8 * c + 4 * half;
        if (d < g.a.dim) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = to_f32(v[d + e]);
            if (sees && !(fabsf(x) < __builtin_inff())) r.o[blk][4 * c + e] += x;
          }
        }
        asm volatile("" ::: "memory");  // one load at a time: this path is rare, its registers are not
      }
  }
}

// A row's results: to the output where the worker had all its units, else to its part.
template <typename T, int DB>
__device__ __forceinline__ void rows_end(const TileArgs& g, const Place& p, int row0, Rows<T, DB>& r, float* part) {
  using S = Shape<T, DB>;
  const int lane = threadIdx.x & 63, half = lane >> 5, row = row0 + (lane & 31);
  const float l = both_halves(r.l);
  if (!r.live) return;
  if (part != nullptr) {
    float* x = part + (int64_t)row * (DB + 2);
#pragma unroll
    for (int b = 0; b < S::kBlocks; ++b)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        typedef float f32x2_u __attribute__((ext_vector_type(2), aligned(8)));
        *reinterpret_cast<f32x2_u*>(x + 32 * b + 8 * (i / 4) + 4 * half + i % 4) = f32x2_u{r.o[b][i], r.o[b][i + 1]};
      }
    if (half == 0) {
      x[DB] = r.m;
      x[DB + 1] = l;
    }
    return;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int i = (uint32_t)row / (uint32_t)g.group;
  T* out = static_cast<T*>(g.a.out) + (p.s.first + p.t * g.per_tile + i) * g.a.o_st +
           (int64_t)(p.h * g.group + (row - i * g.group)) * g.a.o_sh;
#pragma unroll
  for (int b = 0; b < S::kBlocks; ++b)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int d = 32 * b + 8 * c + 4 * half;
      if (d >= g.a.dim) continue;
      const float x0 = r.o[b][4 * c] * inv, x1 = r.o[b][4 * c + 1] * inv, x2 = r.o[b][4 * c + 2] * inv, x3 = r.o[b][4 * c + 3] * inv;
      if constexpr (sizeof(T) == 2) *reinterpret_cast<u32x2*>(out + d) = u32x2{pack2<T>(x0, x1), pack2<T>(x2, x3)};
      else *reinterpret_cast<f32x4_v*>(out + d) = f32x4_v{x0, x1, x2, x3};
    }
}

// The job that a worker leaves, given the part of its last tile that it has begun but not ended (or none).
__device__ __forceinline__ void leave_job(const TileArgs& g, int64_t worker, const Place* p, int64_t slot, int64_t total, int64_t n) {
  Job j{};
  if (p != nullptr) {
    const int t0 = p->t * g.per_tile;
    j.token = p->s.first + t0;
    j.first = slot;
    j.head = p->h * g.group;
    j.rows = min(g.per_tile, p->s.count - t0) * g.group;
    j.parts = (int)(worker_of(p->begin + (p->k.u1 - p->k.u0) - 1, total, n) - worker) + 1;
  }
  g.jobs[worker] = j;
}

// Zeros for the rows of no sequence, a token a wave at a time.
template <typename T>
__device__ __forceinline__ void zero_other_rows(const TileArgs& g, int64_t wave, int64_t waves) {
  const Sequences& s = g.a.seq;
  if (!g.a.zero_other || s.starts == nullptr || (s.starts[0] <= 0 && s.starts[s.batch] >= s.tokens)) return;
  const int lane = threadIdx.x & 63;
  for (int64_t t = wave; t < s.tokens; t += waves) {
    if (sequence_of(s, t) >= 0) continue;
    T* out = static_cast<T*>(g.a.out) + t * g.a.o_st;
    for (int h = 0; h < g.a.q_heads; ++h)
      for (int d = lane; d < g.a.dim; d += 64) out[h * g.a.o_sh + d] = from_f32<T>(0.0f);
  }
}

// The pages of a unit's keys, a key a lane (its 32 or 64 rows): looked up while the unit
// before it is loaded.
template <int UNIT, int GROUP>
struct Pages {
  int page, slot;  // page -1: no key of the tile

  // GROUP rows are loaded together, seen by some row of the tile or not.
  __device__ __forceinline__ void look_up(const TileArgs& g, const Place& p, int key0) {
    const int key = key0 + (threadIdx.x & (UNIT - 1));
    page = -1;
    slot = 0;
    if (key >= (p.k.lo & -GROUP) && key < p.k.hi) {
      uint32_t at, in;
      key_place(g, (uint32_t)key, at, in);
      slot = (int)in;
      page = g.a.pages[p.b * g.a.ld_pages + at];
    }
  }
  __device__ __forceinline__ bool there(const TileArgs& g, int pg) const { return pg >= 0 && pg < (int)g.a.n_pages; }
  // The keys that are there, by row.
  __device__ __forceinline__ uint64_t seen(const TileArgs& g) const {
    const uint64_t all = __ballot(there(g, page));
    return UNIT == 64 ? all : all & 0xFFFFFFFFu;
  }
};

// The K and V rows of a unit, as N loads of a wave each: load i takes rows first + i *
// stride .. + kPerLoad - 1. LANE: pages that are no multiple of a load's rows, so that a
// load's rows are on pages of their own; else its address is scalar work.
template <typename T, int DB, int N, int UNIT, bool LANE>
struct Loads {
  using S = Shape<T, DB>;
  using P = Pages<UNIT, LANE ? 1 : S::kPerLoad>;
  u32x4 k[N], v[N];

  __device__ __forceinline__ void issue(const TileArgs& g, const Place& p, const P& pg, int first, int stride) {
    const int lane = threadIdx.x & 63;
    const int in = lane / S::kChunks, d = (lane % S::kChunks) * S::VE;
    const T* k0 = static_cast<const T*>(g.a.k) + (int64_t)p.h * g.a.kh;
    const T* v0 = static_cast<const T*>(g.a.v) + (int64_t)p.h * g.a.vh;
    if constexpr (LANE) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int page = __shfl(pg.page, first + i * stride + in), slot = __shfl(pg.slot, first + i * stride + in);
        k[i] = v[i] = u32x4{0, 0, 0, 0};
        if (pg.there(g, page) && d < g.a.dim) {
          k[i] = *reinterpret_cast<const u32x4*>(k0 + (int64_t)page * g.a.kp + (int64_t)slot * g.a.ks + d);
          v[i] = *reinterpret_cast<const u32x4*>(v0 + (int64_t)page * g.a.vp + (int64_t)slot * g.a.vs + d);
        }
      }
    } else {
      const int64_t ko = (int64_t)in * g.a.ks + d, vo = (int64_t)in * g.a.vs + d;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        // (rows of the load past the tile's keys are memory of the same page, hidden below)
        const int page = __builtin_amdgcn_readlane(pg.page, first + i * stride);
        const int slot = __builtin_amdgcn_readlane(pg.slot, first + i * stride);
        k[i] = v[i] = u32x4{0, 0, 0, 0};
        if (pg.there(g, page) && d < g.a.dim) {
          k[i] = *reinterpret_cast<const u32x4*>(k0 + ((int64_t)page * g.a.kp + (int64_t)slot * g.a.ks) + ko);
          v[i] = *reinterpret_cast<const u32x4*>(v0 + ((int64_t)page * g.a.vp + (int64_t)slot * g.a.vs) + vo);
        }
      }
    }
  }

  // Into LDS. edge: the unit holds keys outside the tile's, whose values become 0; clean:
  // values that are not finite do, too. Returns whether this lane had some.
  __device__ __forceinline__ bool store(const Place& p, int key0, int first, int stride, char* kl, char* vl, bool edge, bool clean) {
    const int lane = threadIdx.x & 63;
    const int in = lane / S::kChunks, chunk = lane % S::kChunks;
    uint32_t found = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int row = first + i * stride + in;
      if (edge && (key0 + row < p.k.lo || key0 + row >= p.k.hi)) v[i] = u32x4{0, 0, 0, 0};
      if (clean) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t bad = not_finite<T>(v[i][e]);
          found |= bad;
          v[i][e] = finite_only<T>(v[i][e], bad);
        }
      }
      *reinterpret_cast<u32x4*>(kl + row * S::kPitch + 16 * chunk) = k[i];
      *reinterpret_cast<u32x4*>(vl + row * S::vPitch + 16 * chunk) = v[i];
    }
    return found != 0;
  }
};

// The next tile of the line after p.
__device__ __forceinline__ void next_place(const TileArgs& g, Place& p) {
  p.begin += p.k.u1 - p.k.u0;
  if (++p.t == tiles_of(g, p.s)) {
    p.t = 0;
    if (++p.h == g.a.kv_heads) {
      p.h = 0;
      do {
        ++p.b;
        p.s = seq_at(g, p.b);
      } while (p.s.count == 0 && p.b + 1 < g.a.seq.batch);
    }
  }
  p.k = span_of(g, p.s, p.t);
}

// ---------------------------------------------------------------------------
// Few rows: a wave is a worker
// ---------------------------------------------------------------------------
constexpr int kFewWaves = 4;

template <typename T, int DB, bool LANE>
__global__ void __launch_bounds__(64 * kFewWaves, DB * sizeof(T) <= 256 ? 2 : 1) attend_few_kernel(TileArgs g, bool lined) {
  using S = Shape<T, DB>;
  constexpr int N = 32 / S::kPerLoad;
  __shared__ __attribute__((aligned(16))) char lds[kFewWaves][32 * (S::kPitch + S::vPitch)];
  __shared__ int64_t sums[kFewWaves];
  __shared__ int64_t found[kFewWaves][3];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t worker = (int64_t)blockIdx.x * kFewWaves + wave;
  const int64_t batch = g.a.seq.batch;
  int64_t total, n_workers, u0, u1, at = 0, units = 0;
  Place p;
  if (lined) {
    total = g.line[batch];
    n_workers = active_workers(g, total);
    u0 = begin_of(worker, total, n_workers);
    if (total > 0 && worker < n_workers) {
      p.b = sequence_at(g.line, batch, u0);
      at = g.line[p.b];
      units = g.line[p.b + 1] - at;
    }
  } else {
    // every workgroup lines the sequences up: 4 a thread, at most
    int64_t mine[kPlanBatch / (64 * kFewWaves)], sum = 0;
#pragma unroll
    for (int i = 0; i < kPlanBatch / (64 * kFewWaves); ++i) {
      const int64_t b = (int64_t)threadIdx.x * (kPlanBatch / (64 * kFewWaves)) + i;
      mine[i] = b < batch ? units_of(g, seq_at(g, b), 0, 1) * g.a.kv_heads : 0;
      sum += mine[i];
    }
    int64_t upto = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t o = __shfl_up(upto, d);
      if (lane >= d) upto += o;
    }
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    total = 0;
    int64_t before = upto - sum;
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) {
      if (w < wave) before += sums[w];
      total += sums[w];
    }
    n_workers = active_workers(g, total);
#pragma unroll
    for (int i = 0; i < kPlanBatch / (64 * kFewWaves); ++i) {
      const int64_t b = (int64_t)threadIdx.x * (kPlanBatch / (64 * kFewWaves)) + i;
      for (int w = 0; w < kFewWaves; ++w) {
        const int64_t x = begin_of((int64_t)blockIdx.x * kFewWaves + w, total, n_workers);
        if (x >= before && x < before + mine[i]) {
          found[w][0] = b;
          found[w][1] = before;
          found[w][2] = mine[i];
        }
      }
      before += mine[i];
    }
    __syncthreads();
    u0 = begin_of(worker, total, n_workers);
    p.b = found[wave][0];
    at = found[wave][1];
    units = found[wave][2];
  }
  zero_other_rows<T>(g, worker, (int64_t)gridDim.x * kFewWaves);
  if (total == 0 || worker >= n_workers) {
    if (lane == 0) leave_job(g, worker, nullptr, 0, 0, 0);
    return;
  }
  u1 = begin_of(worker + 1, total, n_workers);
  p.b = ((int64_t)__builtin_amdgcn_readfirstlane((int)(p.b >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)p.b);
  place_in_sequence(g, p, u0, at, units);
  const int64_t first_begin = p.begin;

  char* kl = lds[wave];
  char* vl = lds[wave] + 32 * S::kPitch;
  Loads<T, DB, N, 32, LANE> x;
  typename Loads<T, DB, N, 32, LANE>::P pg;
  Rows<T, DB> r;
  for (int64_t u = u0; u < u1;) {
    const int64_t tile_end = p.begin + (p.k.u1 - p.k.u0);
    const int64_t stop = min(tile_end, u1);
    const bool whole = u == p.begin && stop == tile_end;
    const int tokens = min(g.per_tile, p.s.count - p.t * g.per_tile);
    int key0 = __builtin_amdgcn_readfirstlane((p.k.u0 + (int)(u - p.begin)) * 32);
    const int key1 = __builtin_amdgcn_readfirstlane(key0 + 32 * (int)(stop - u));
    pg.look_up(g, p, key0);
    rows_begin<T, DB>(g, p, 0, r);
    x.issue(g, p, pg, 0, S::kPerLoad);
    uint32_t next = (uint32_t)pg.seen(g);
    pg.look_up(g, p, key0 + 32);
    for (; key0 < key1; key0 += 32) {
      const uint32_t seen = next;
      const bool edge = key0 < p.k.lo || key0 + 32 > p.k.hi;
      const bool mask = key0 < r.low || key0 + 32 > r.top || seen != 0xFFFFFFFFu;
      const bool bad = x.store(p, key0, 0, S::kPerLoad, kl, vl, edge, mask && tokens > 1);
      if (key0 + 32 < key1) {
        x.issue(g, p, pg, 0, S::kPerLoad);
        next = (uint32_t)pg.seen(g);
        pg.look_up(g, p, key0 + 64);
      }
      f32x16_t s[1];
      s[0] = scores32<T, DB>(g, r, kl, 0);
      if (mask) hide32<T, DB>(r, s[0], key0, seen);
      new_maximum<T, DB, 1>(g, r, s);
      weights32<T, DB>(g, r, s[0]);
      values32<T, DB>(r, s[0], vl, 0);
      if (__any(bad)) add_not_finite<T, DB>(g, p, r, key0, seen);
    }
    u = stop;
    float* part = nullptr;
    const int64_t slot = 2 * worker + (p.begin != first_begin);
    if (!whole) part = g.part + slot * g.rows * (DB + 2);
    rows_end<T, DB>(g, p, 0, r, part);
    if (u < u1) next_place(g, p);
    else if (lane == 0) leave_job(g, worker, p.begin >= u0 && !whole ? &p : nullptr, slot, total, n_workers);
  }
}

// ---------------------------------------------------------------------------
// Many rows: a workgroup is a worker, its waves share the units' keys and values
// ---------------------------------------------------------------------------
template <typename T, int DB, int WAVES, int UNIT, bool LANE>
__global__ void __launch_bounds__(64 * WAVES) attend_many_kernel(TileArgs g) {
  using S = Shape<T, DB>;
  constexpr int N = UNIT / S::kPerLoad / WAVES;  // loads of a wave, UNIT rows over all waves
  static_assert(N >= 1 && N * S::kPerLoad * WAVES == UNIT, "a unit is whole loads of every wave");
  constexpr int kV = UNIT * S::kPitch;
  __shared__ __attribute__((aligned(16))) char lds[2][UNIT * (S::kPitch + S::vPitch)];  // two units' K and V
  __shared__ uint32_t bad[2];  // the unit (by count) whose values are not all finite
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // neighbours in the line, which share keys, go to one XCD
  const int64_t nb = gridDim.x;
  const int64_t worker = nb % 8 == 0 ? (int64_t)(blockIdx.x % 8) * (nb / 8) + blockIdx.x / 8 : blockIdx.x;
  const int64_t total = g.line[g.a.seq.batch];
  const int64_t n_workers = active_workers(g, total);
  zero_other_rows<T>(g, worker * WAVES + wave, nb * WAVES);
  if (total == 0 || worker >= n_workers) {
    if (threadIdx.x == 0) leave_job(g, worker, nullptr, 0, 0, 0);
    return;
  }
  const int64_t u0 = begin_of(worker, total, n_workers), u1 = begin_of(worker + 1, total, n_workers);
  Place p;
  p.b = sequence_at(g.line, g.a.seq.batch, u0);
  const int64_t at = g.line[p.b];
  place_in_sequence(g, p, u0, at, g.line[p.b + 1] - at);
  const int64_t first_begin = p.begin;
  const int row0 = wave * kRows, first = wave * S::kPerLoad;
  constexpr int stride = WAVES * S::kPerLoad;
  if (threadIdx.x < 2) bad[threadIdx.x] = 0;
  __syncthreads();

  Loads<T, DB, N, UNIT, LANE> x;
  typename Loads<T, DB, N, UNIT, LANE>::P pg;
  Rows<T, DB> r;
  int buf = 0;
  uint32_t serial = 0;
  for (int64_t u = u0; u < u1;) {
    const int64_t tile_end = p.begin + (p.k.u1 - p.k.u0);
    const int64_t stop = min(tile_end, u1);
    const bool whole = u == p.begin && stop == tile_end;
    const int t0 = p.t * g.per_tile, tokens = min(g.per_tile, p.s.count - t0);
    int key0 = __builtin_amdgcn_readfirstlane((p.k.u0 + (int)(u - p.begin)) * UNIT);
    const int key1 = __builtin_amdgcn_readfirstlane(key0 + UNIT * (int)(stop - u));
    pg.look_up(g, p, key0);
    rows_begin<T, DB>(g, p, row0, r);
    // the keys that some row of this wave sees (none without rows), and that every row of the tile does
    const int w0 = row0 / g.group, w1 = min((row0 + kRows - 1) / g.group, tokens - 1);
    const int end = w0 < tokens ? __builtin_amdgcn_readfirstlane(min(p.s.pos0 + t0 + w1 + 1, p.s.length)) : 0;
    const int all_top = __builtin_amdgcn_readfirstlane(p.s.pos0 + t0 + 1);
    int beg = 0, all_low = 0;
    if (g.a.window > 0) {
      beg = __builtin_amdgcn_readfirstlane((int)max((int64_t)p.s.pos0 + t0 + w0 + 1 - g.a.window, (int64_t)0));
      all_low = __builtin_amdgcn_readfirstlane((int)max((int64_t)p.s.pos0 + t0 + tokens - g.a.window, (int64_t)0));
    }
    auto put = [&](int key, int to) {
      const bool edge = key < p.k.lo || key + UNIT > p.k.hi;
      const bool clean = tokens > 1 && (key < all_low || key + UNIT > all_top);
      ++serial;
      if (x.store(p, key, first, stride, lds[to], lds[to] + kV, edge, clean)) bad[to] = serial;
    };
    x.issue(g, p, pg, first, stride);
    uint64_t next = pg.seen(g);
    pg.look_up(g, p, key0 + UNIT);
    put(key0, buf);
    __syncthreads();
    for (; key0 < key1; key0 += UNIT, buf ^= 1) {
      const bool more = key0 + UNIT < key1;
      const uint64_t seen = next;
      const uint32_t now = serial;
      if (more) {
        x.issue(g, p, pg, first, stride);
        next = pg.seen(g);
        pg.look_up(g, p, key0 + 2 * UNIT);
      }
      if (key0 < end && key0 + UNIT > beg) {
#pragma unroll
        for (int n = 0; n < UNIT / 32; ++n) {
          const int key = key0 + 32 * n;
          if (n > 0 && key >= end) break;
          const uint32_t bits = (uint32_t)(seen >> (32 * n));
          f32x16_t s[1];
          s[0] = scores32<T, DB>(g, r, lds[buf], 32 * n);
          if (key < r.low || key + 32 > r.top || bits != 0xFFFFFFFFu) hide32<T, DB>(r, s[0], key, bits);
          new_maximum<T, DB, 1>(g, r, s);
          weights32<T, DB>(g, r, s[0]);
          values32<T, DB>(r, s[0], lds[buf] + kV, 32 * n);
          if (__builtin_amdgcn_readfirstlane(bad[buf]) == now) add_not_finite<T, DB>(g, p, r, key, bits);
        }
      }
      if (more) put(key0 + UNIT, buf ^ 1);
      __syncthreads();
    }
    u = stop;
    float* part = nullptr;
    const int64_t slot = 2 * worker + (p.begin != first_begin);
    if (!whole) part = g.part + slot * g.rows * (DB + 2);
    rows_end<T, DB>(g, p, row0, r, part);
    if (u < u1) next_place(g, p);
    else if (threadIdx.x == 0) leave_job(g, worker, p.begin >= u0 && !whole ? &p : nullptr, slot, total, n_workers);
  }
}

// ---------------------------------------------------------------------------
// Joining the parts: a job for each worker whose last tile goes on in the next one
// ---------------------------------------------------------------------------
template <typename T, int DB>
__global__ void __launch_bounds__(256) attend_join_kernel(TileArgs g) {
  constexpr int kVals = DB / 64;
  __shared__ float sums[4][DB];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Job job = g.jobs[blockIdx.x];
  const int rows = job.rows, parts = job.parts;
  if (rows == 0) return;
  const int64_t one = (int64_t)g.rows * (DB + 2);
  const float* first = g.part + job.first * one;
  const float* rest = g.part + 2 * ((int64_t)blockIdx.x + 1) * one;  // part i > 0: two slots further each
  auto part = [&](int i, int row) { return (i == 0 ? first : rest + (int64_t)(i - 1) * 2 * one) + (int64_t)row * (DB + 2); };
  auto store = [&](int row, const float* acc, float inv) {
    const int i = (uint32_t)row / (uint32_t)g.group;
    T* out = static_cast<T*>(g.a.out) + (job.token + i) * g.a.o_st + (int64_t)(job.head + row - i * g.group) * g.a.o_sh;
#pragma unroll
    for (int v = 0; v < kVals; ++v)
      if (64 * v + lane < g.a.dim) out[64 * v + lane] = from_f32<T>(acc[v] * inv);
  };
  typedef float f32x2_a __attribute__((ext_vector_type(2), aligned(8)));
  const auto factor = [](float m, float top) { return top == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(m - top); };
  if (parts <= 8) {
    // R rows a wave, their loads together; a row's maxima and sums in every lane
    constexpr int R = 4;
    for (int row0 = (blockIdx.y * 4 + wave) * R; row0 < rows; row0 += 4 * R * gridDim.y) {
      float top[R], sum[R], acc[R][kVals];
#pragma unroll
      for (int k = 0; k < R; ++k) {
        top[k] = kNegInf;
        sum[k] = 0.0f;
#pragma unroll
        for (int v = 0; v < kVals; ++v) acc[k][v] = 0.0f;
      }
      for (int i = 0; i < parts; ++i) {
        f32x2_a ml[R];
        float x[R][kVals];
#pragma unroll
        for (int k = 0; k < R; ++k) {
          const float* src = part(i, min(row0 + k, rows - 1));
          ml[k] = *reinterpret_cast<const f32x2_a*>(src + DB);
#pragma unroll
          for (int v = 0; v < kVals; ++v) x[k][v] = src[64 * v + lane];
        }
#pragma unroll
        for (int k = 0; k < R; ++k) {
          const float now = fmaxf(top[k], ml[k][0]), keep = factor(top[k], now), f = factor(ml[k][0], now);
          top[k] = now;
          sum[k] = sum[k] * keep + ml[k][1] * f;
#pragma unroll
          for (int v = 0; v < kVals; ++v) acc[k][v] = acc[k][v] * keep + x[k][v] * f;
        }
      }
#pragma unroll
      for (int k = 0; k < R; ++k)
        if (row0 + k < rows) store(row0 + k, acc[k], sum[k] == 0.0f ? 0.0f : 1.0f / sum[k]);
    }
    return;
  }
  // many parts: a row at a time, its parts over the waves
  for (int row = blockIdx.y; row < rows; row += gridDim.y) {
    float top = kNegInf, sum = 0.0f, acc[kVals] = {};
    for (int i = lane; i < parts; i += 64) top = fmaxf(top, part(i, row)[DB]);
    top = wave_max(top);
    for (int i = lane; i < parts; i += 64) sum += factor(part(i, row)[DB], top) * part(i, row)[DB + 1];
    sum = wave_sum(sum);
#pragma unroll 8
    for (int i = wave; i < parts; i += 4) {
      const float* x = part(i, row);
      const float f = factor(x[DB], top);
#pragma unroll
      for (int v = 0; v < kVals; ++v) acc[v] = fmaf(f, x[64 * v + lane], acc[v]);
    }
#pragma unroll
    for (int v = 0; v < kVals; ++v) sums[wave][64 * v + lane] = acc[v];
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int v = 0; v < kVals; ++v) {
        const int d = 64 * v + lane;
        acc[v] = (sums[0][d] + sums[1][d]) + (sums[2][d] + sums[3][d]);
      }
      store(row, acc, sum == 0.0f ? 0.0f : 1.0f / sum);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
struct Plan {
  bool few, lined, cut;
  int padded, waves, unit, per_tile, rows, min_units;
  int64_t workers;
  size_t line_bytes, job_bytes, part_bytes;
};

Plan plan_of(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t max_keys, int64_t max_chunk,
             int dtype) {
  Plan p{};
  const bool f32 = dtype == AK_DTYPE_F32;
  const int64_t group = q_heads / kv_heads;
  p.padded = dim <= 64 ? 64 : dim <= 128 ? 128 : 256;
  max_chunk = std::min(max_chunk, tokens);
  const bool wide = p.padded * (f32 ? 4 : 2) > 256;  // rows past 256 bytes: half the waves and keys
  p.few = max_chunk * group <= kRows && p.padded < 256;
  p.waves = p.few || wide ? 4 : 8;
  p.unit = p.few || wide ? 32 : 64;
  const int64_t rows = p.few ? kRows : kRows * p.waves;
  p.per_tile = (int)std::max((int64_t)1, std::min(rows / group, max_chunk));
  p.rows = (int)(p.per_tile * group);
  p.min_units = p.few ? 4 : 2;
  // (many tiles of a sequence are lined up by 64 lanes: an understated max_chunk)
  p.lined = !p.few || batch > kPlanBatch || tokens / p.per_tile > batch + 4096;
  // workgroups at once: two of the few-row kernel where their LDS and registers leave room
  const int64_t groups = (int64_t)cu_count() * (p.few && !wide ? 2 : 1);
  const double most = (double)kv_heads * ((double)tokens / p.per_tile + (double)batch) * ((double)max_keys / p.unit + 1.0);
  const int64_t useful = most > 1e9 ? (int64_t)1 << 30 : (int64_t)most / p.min_units + 1;
  p.workers = std::min(groups * (p.few ? kFewWaves : 1), useful);
  if (p.few) p.workers = (p.workers + kFewWaves - 1) / kFewWaves * kFewWaves;
  p.cut = p.workers > 8 * kv_heads * (tokens / p.per_tile);
  p.line_bytes = (size_t)(batch + 2) / 2 * 16;
  p.job_bytes = (size_t)p.workers * sizeof(Job);
  p.part_bytes = (size_t)p.workers * 2 * (size_t)p.rows * (size_t)(p.padded + 2) * sizeof(float);
  return p;
}

template <typename T, int DB, bool LANE>
void launch_tiles(const TileArgs& g, const Plan& p, hipStream_t s) {
  if (p.lined) attend_line_kernel<<<dim3(1), dim3(1024), 0, s>>>(g);
  if constexpr (DB < 256) {
    if (p.few) attend_few_kernel<T, DB, LANE><<<dim3((unsigned)(p.workers / kFewWaves)), dim3(64 * kFewWaves), 0, s>>>(g, p.lined);
  }
  if (!p.few) {
    constexpr int kWaves = DB * sizeof(T) > 256 ? 4 : 8, kUnit = DB * sizeof(T) > 256 ? 32 : 64;
    attend_many_kernel<T, DB, kWaves, kUnit, LANE><<<dim3((unsigned)p.workers), dim3(64 * kWaves), 0, s>>>(g);
  }
  if (p.workers > 1) {
    // (of few rows in many parts a row a workgroup, of many rows 16)
    const unsigned slices = (unsigned)(p.rows > kRows ? (p.rows + 15) / 16 : p.cut ? std::min(p.rows, 4) : 1);
    attend_join_kernel<T, DB><<<dim3((unsigned)(p.workers - 1), slices), dim3(256), 0, s>>>(g);
  }
}

template <typename T>
void launch_type(TileArgs& g, const Plan& p, hipStream_t s) {
  auto go = [&](auto db) {
    constexpr int DB = decltype(db)::value;
    if (g.a.page_size % Shape<T, DB>::kPerLoad) launch_tiles<T, DB, true>(g, p, s);
    else launch_tiles<T, DB, false>(g, p, s);
  };
  if (p.padded == 64) go(std::integral_constant<int, 64>());
  else if (p.padded == 128) go(std::integral_constant<int, 128>());
  else go(std::integral_constant<int, 256>());
}

}  // namespace

bool attend_tiles_take(const AttendArgs& a, int dtype) {
  const int ve = 16 / ak_dtype_size(dtype);
  const int64_t group = a.q_heads / a.kv_heads;
  bool ok = a.dim <= 256 && a.dim % ve == 0 && group <= kRows * (a.dim > 128 || (a.dim > 64 && ve == 4) ? 4 : 8);
  for (const void* x : {a.q, a.k, a.v, (const void*)a.out}) ok = ok && aligned16(x);
  for (int64_t st : {a.q_st, a.q_sh, a.o_st, a.o_sh, a.kp, a.ks, a.kh, a.vp, a.vs, a.vh}) ok = ok && st % ve == 0;
  return ok;
}

size_t attend_tiles_workspace_bytes(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim,
                                    int64_t max_keys, int64_t max_chunk, int dtype) {
  const Plan p = plan_of(tokens, batch, q_heads, kv_heads, dim, max_keys, max_chunk, dtype);
  return p.line_bytes + p.job_bytes + p.part_bytes;
}

void attend_tiles(const AttendArgs& a, int64_t max_chunk, int dtype, void* workspace, hipStream_t s) {
  const Plan p = plan_of(a.seq.tokens, a.seq.batch, a.q_heads, a.kv_heads, a.dim, a.max_pages * a.page_size, max_chunk, dtype);
  TileArgs g{};
  g.a = a;
  g.group = a.q_heads / a.kv_heads;
  g.per_tile = p.per_tile;
  g.page_magic = (uint32_t)std::min(((uint64_t)1 << 32) / (uint64_t)a.page_size, (uint64_t)UINT32_MAX);
  g.unit = p.unit;
  g.rows = p.rows;
  g.workers = (int)p.workers;
  g.min_units = p.min_units;
  g.line = static_cast<int64_t*>(workspace);
  g.jobs = reinterpret_cast<Job*>(static_cast<char*>(workspace) + p.line_bytes);
  g.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.line_bytes + p.job_bytes);
  if (a.softcap > 0.0f) {
    g.cap_in = a.scale / a.softcap;
    g.cap_out = a.softcap * kLog2e;
    g.c = 1.0f;
  } else {
    g.c = a.scale * kLog2e;
  }
  if (dtype == AK_DTYPE_F32) launch_type<float>(g, p, s);
  else if (dtype == AK_DTYPE_F16) launch_type<f16>(g, p, s);
  else launch_type<bf16>(g, p, s);
}

}  // namespace ak
