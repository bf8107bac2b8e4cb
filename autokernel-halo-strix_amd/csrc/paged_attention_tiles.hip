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
constexpr int kPlanBatch = 1024;   // sequences that a workgroup of few-row workers lines up by itself,
constexpr int kPlanMany = 64;      // and one of many rows, a wave a sequence (a launch for it: 3 us more of 17 to 25)

typedef float f32x4_v __attribute__((ext_vector_type(4)));

// What the joining kernel does for a worker: the rows of its last tile, whose first part
// is the worker's own.
struct Job {
  int64_t first;         // the part's slot
  int token, head;       // the tile's first token of the call, its first query head
  int rows, parts;       // rows 0: nothing
};

struct TileArgs {
  AttendArgs a;
  int group, per_tile;             // heads of a group, tokens of a tile
  uint32_t page_magic;             // floor(2^32 / page_size), at most 2^32 - 1
  int unit, rows;                  // keys of a unit, rows of a tile
  int workers, min_units;
  uint32_t kp, ks, vp, vs;         // cache strides in bytes: page, slot
  float join_cost;                 // of a part, in a unit's time, over the number of tiles
  int64_t* line;                   // [batch + 1]: the units before each sequence
  Job* jobs;                       // [workers]
  float* part;                     // [2 workers]: sums of products, maxima, sums of a tile's rows
  float c, cap_in, cap_out;        // exponents in base 2: c s; cap_in > 0: c cap(s), see cap32
  float unit2;                     // the references' unit as an exponent in base 2: 1, or c, see Reference
};

// The kernels' argument where the launch left it. Held in registers all of it would crowd
// out what the loops need (100 scalars went through vector registers there, a quarter of the
// instructions): what a tile's ends need is read anew for each, through fresh().
typedef const TileArgs __attribute__((address_space(4)))* Args;

__device__ __forceinline__ Args kernel_args() { return (Args)__builtin_amdgcn_kernarg_segment_ptr(); }
__device__ __forceinline__ Args fresh(Args g) {
  asm volatile("" : "+s"(g));
  return g;
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform64(int64_t v) {
  return (int64_t)((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32 | (uint32_t)uniform((int)v));
}

// Where a key lives.
struct PageMath {
  uint32_t size, magic;
  __device__ __forceinline__ void place(uint32_t key, uint32_t& page, uint32_t& slot) const {
    page = __umulhi(key, magic);  // the quotient or one less
    slot = key - page * size;
    if (slot >= size) {
      slot -= size;
      ++page;
    }
  }
};
__device__ __forceinline__ PageMath page_math(Args g) { return {(uint32_t)g->a.page_size, g->page_magic}; }

// A sequence's part in the line.
struct Seq {
  int first, count;   // its new tokens
  int length, pos0;   // positions that can have keys, position of the first new token
};

__device__ __forceinline__ Seq seq_at(Args g, int b) {
  Seq s;
  const int tokens = (int)g->a.seq.tokens;
  int64_t count;
  if (g->a.seq.starts == nullptr) {
    s.first = b * (int)g->a.seq.per;
    count = g->a.seq.per;
  } else {
    const int a = g->a.seq.starts[b], e = g->a.seq.starts[b + 1];
    s.first = min(max(a, 0), tokens);
    count = max(min(e, tokens) - s.first, 0);
  }
  const int length = g->a.seq.lengths[b];
  s.count = (int)count;
  // (far below 0 all the same once it is: no key)
  s.pos0 = (int)max((int64_t)length - count, (int64_t)INT32_MIN / 2);
  s.length = (int)min((int64_t)length, g->a.max_pages * g->a.page_size);
  return s;
}

// The keys [lo, hi) that some token of tile t sees, in units [u0, u1) (one at least).
struct Span {
  int lo, hi, u0, u1;
};

__device__ __forceinline__ Span span_of(Args g, const Seq& s, int t) {
  const int t0 = t * g->per_tile, t1 = min(t0 + g->per_tile, s.count);
  Span r;
  r.hi = max(min(s.pos0 + t1, s.length), 0);
  r.lo = 0;
  if (g->a.window > 0) r.lo = (int)min(max((int64_t)s.pos0 + t0 + 1 - g->a.window, (int64_t)0), (int64_t)r.hi);
  r.u0 = (uint32_t)r.lo / (uint32_t)g->unit;
  r.u1 = max((int)(((uint32_t)r.hi + g->unit - 1) / (uint32_t)g->unit), r.u0 + 1);
  return r;
}

__device__ __forceinline__ int tiles_of(Args g, const Seq& s) { return (s.count + g->per_tile - 1) / g->per_tile; }

// Workers that a line of `total` units keeps busy; worker w has [begin(w), begin(w + 1)). A
// tile of n units takes n / parts of a unit's time and then parts times join_cost of it to be
// joined, least at units of sqrt(n join_cost) a part: 7 tokens over 69571 keys of one head took
// 226 us with a worker a unit, so 35; 4 tokens over 20284 keys 160 and 31.
__device__ __forceinline__ int64_t active_workers(Args g, int64_t total) {
  const int64_t least = max((int64_t)g->min_units, (int64_t)sqrtf((float)total * g->join_cost));
  return max(min((int64_t)g->workers, total / least), (int64_t)1);
}
__device__ __forceinline__ int64_t begin_of(int64_t w, int64_t total, int64_t n) { return w * total / n; }
__device__ __forceinline__ int64_t worker_of(int64_t u, int64_t total, int64_t n) { return ((u + 1) * n - 1) / total; }

__device__ __forceinline__ int64_t wave_sum64(int64_t v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

// A tile of the line, and which of its units come first and end (a worker's share of it).
struct Place {
  int b, h, t;     // sequence, key head, tile of the sequence
  Seq s;
  Span k;
};

// The tile of a sequence's unit `rest` (counted from the sequence's first); `rest` becomes
// the unit of the tile. All lanes of a wave together.
__device__ __forceinline__ void place_in_sequence(Args g, Place& p, int64_t& rest, int64_t units) {
  const int lane = threadIdx.x & 63;
  p.s = seq_at(g, p.b);
  const int64_t each = units / g->a.kv_heads;
  const int h = (int)(rest / each);
  rest -= (int64_t)h * each;
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
  p.t = uniform(t);
  p.h = uniform(h);
  p.k = span_of(g, p.s, p.t);
}

// The tile after p.
__device__ __forceinline__ void next_place(Args g, Place& p) {
  if (++p.t == tiles_of(g, p.s)) {
    p.t = 0;
    if (++p.h == g->a.kv_heads) {
      p.h = 0;
      do {
        ++p.b;
        p.s = seq_at(g, p.b);
      } while (p.s.count == 0 && p.b + 1 < (int)g->a.seq.batch);
      p.s.first = uniform(p.s.first);
      p.s.count = uniform(p.s.count);
      p.s.length = uniform(p.s.length);
      p.s.pos0 = uniform(p.s.pos0);
    }
  }
  p.k = span_of(g, p.s, p.t);
}

// The sequence of unit u from the line in memory: 64 entries at a time.
__device__ __forceinline__ int sequence_at(const int64_t* line, int batch, int64_t u) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = batch;
  while (n > 1) {
    const int step = (n + 63) / 64;
    const bool le = (int64_t)lane * step < n && line[lo + lane * step] <= u;
    const int last = 63 - __builtin_clzll(__ballot(le) | 1);
    const int next = lo + last * step;
    n = min(step, lo + n - next);
    lo = next;
  }
  // (sequences without units begin where the next one does: the last of them is ours)
  return uniform(lo);
}

__device__ __forceinline__ int64_t units_of(Args g, const Seq& s, int first_tile, int step) {
  int64_t sum = 0;
  const int n = tiles_of(g, s);
  for (int t = first_tile; t < n; t += step) {
    const Span k = span_of(g, s, t);
    sum += k.u1 - k.u0;
  }
  return sum;
}

// Lines up the units of all sequences: a wave each, then their sums.
__global__ void __launch_bounds__(1024) attend_line_kernel(TileArgs) {
  __shared__ int64_t sums[16];
  const Args g = kernel_args();
  int64_t* const line = g->line;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t batch = g->a.seq.batch;
  for (int64_t b = wave; b < batch; b += 16) {
    const int64_t n = wave_sum64(units_of(g, seq_at(g, (int)b), lane, 64));
    if (lane == 0) line[b + 1] = n * g->a.kv_heads;
  }
  if (threadIdx.x == 0) line[0] = 0;
  __syncthreads();
  int64_t before = 0;
  for (int64_t b0 = 0; b0 < batch; b0 += 1024) {
    const int64_t b = b0 + threadIdx.x;
    int64_t upto = b < batch ? line[b + 1] : 0;
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
    if (b < batch) line[b + 1] = upto + add;
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
  // Rows in LDS are a chunk (K: a column of chunks is read) or more (V: four chunks of four
  // rows are read together) longer than their values, which spreads them over the banks: four
  // leave V without conflicts, two with one in three reads twice as long, but room for two
  // workgroups of few rows a CU (of many rows prompts 533 us with two, 524 with four).
  static constexpr int kRowBytes = DB * (int)sizeof(T);
  static constexpr int kPitch = kRowBytes + 16, vPitch = kRowBytes + 32, vWidePitch = kRowBytes + 64;
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
  float m, l;     // what the weights are taken beside (the lane's query) and this half's sum
  int lo, hi;     // the keys that the query sees
  int top, low;   // of the wave's rows: the least hi, the largest lo
  int beg, end;   // of the wave's rows: the keys that some of them see
};

// From scores to exponents in base 2 (Reference has the rest).
struct ScoreMath {
  float c, cap_in, cap_out, to_unit, lag;
  bool cap, bare;
};
template <typename T>
__device__ __forceinline__ ScoreMath score_math(Args g);

// Loads the queries of rows [row0, row0 + 32) of a tile.
template <typename T, int DB>
__device__ __forceinline__ void rows_load(Args g0, const Place& p, int row0, Rows<T, DB>& r) {
  using S = Shape<T, DB>;
  const Args g = fresh(g0);
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int t0 = p.t * g->per_tile, tokens = min(g->per_tile, p.s.count - t0), group = g->group, dim = g->a.dim;
  const int row = row0 + (lane & 31);
  const int i = (uint32_t)row / (uint32_t)group;  // token of the tile
  const bool live = i < tokens;
  const T* q = static_cast<const T*>(g->a.q) + (int64_t)(p.s.first + t0 + min(i, tokens - 1)) * g->a.q_st +
               (int64_t)(p.h * group + (row - i * group)) * g->a.q_sh;
#pragma unroll
  for (int k = 0; k < S::kSteps; ++k) {
    r.q[k] = u32x4{0, 0, 0, 0};
    const int d = (2 * k + half) * S::VE;
    if (live && d < dim) r.q[k] = *reinterpret_cast<const u32x4*>(q + d);
  }
}

// Starts the sums of rows [row0, row0 + 32) of a tile.
template <typename T, int DB>
__device__ __forceinline__ void rows_begin(Args g0, const Place& p, int row0, Rows<T, DB>& r) {
  using S = Shape<T, DB>;
  const Args g = fresh(g0);
  const int lane = threadIdx.x & 63;
  const int t0 = p.t * g->per_tile, tokens = min(g->per_tile, p.s.count - t0), group = g->group;
  const int row = row0 + (lane & 31);
  const int i = (uint32_t)row / (uint32_t)group;  // token of the tile
  const bool live = i < tokens;
  const int tok = min(i, tokens - 1);
  const int pos = p.s.pos0 + t0 + tok;
  const int64_t window = g->a.window;
  r.hi = live ? max(min(pos + 1, p.s.length), 0) : 0;
  r.lo = window > 0 ? (int)max((int64_t)pos + 1 - window, (int64_t)0) : 0;
  // (rows past the tile's see what its last token does: nothing of theirs is kept, and they mask nothing)
  const int i0 = (uint32_t)row0 / (uint32_t)group, i1 = min((int)((uint32_t)(row0 + 31) / (uint32_t)group), tokens - 1);
  const int pos_0 = p.s.pos0 + t0 + min(i0, tokens - 1), pos_1 = p.s.pos0 + t0 + i1;
  r.top = uniform(max(min(pos_0 + 1, p.s.length), 0));
  r.end = i0 < tokens ? uniform(min(pos_1 + 1, p.s.length)) : 0;
  r.low = r.beg = 0;
  if (window > 0) {
    r.low = uniform((int)max((int64_t)pos_1 + 1 - window, (int64_t)0));
    r.beg = uniform((int)max((int64_t)pos_0 + 1 - window, (int64_t)0));
  }
#pragma unroll
  for (int b = 0; b < S::kBlocks; ++b) r.o[b] = f32x16_t{};
  r.m = kNegInf;
  r.l = 0.0f;
}

// Scores of the 32 keys whose K is at row0 on in LDS.
template <typename T, int DB>
__device__ __forceinline__ f32x16_t scores32(const Rows<T, DB>& r, const char* kl, int row0) {
  using S = Shape<T, DB>;
  const int lane = threadIdx.x & 63, half = lane >> 5, row = row0 + (lane & 31);
  const char* base = kl + row * S::kPitch + 16 * half;
  f32x16_t s{};
#pragma unroll
  for (int k = 0; k < S::kSteps; ++k) s = mfma_step(T(), *reinterpret_cast<const u32x4*>(base + 32 * k), r.q[k], s);
  return s;
}

// Capped scores. Of 16-bit types and caps up to kQuickCap: softcap tanh(x) is softcap -
// 2 softcap / (exp(2 x) + 1), whose first term a softmax does not see. Its error of up to
// 4 softcap 2^-24 is absolute, 2^-14 at most, a quarter of a weight's rounding. (16 sequences of
// up to 7000 keys, chunks of up to 500 tokens, 32 + 8 heads of 128: 361 us, with tanh_f32 458
// (each beside the other).) Beyond, fp16 and fp32 take cap_tanh, whose error is relative to the
// score; bf16 tanh_f32, whose error of up to softcap 2^-24 is a third of its weights' rounding at
// the largest cap (prompts of 4 x 2048 tokens, 32 + 8 heads of 128, 287 us, with cap_tanh 348).
constexpr float kQuickCap = 256.0f;

template <typename T>
__device__ __forceinline__ void cap32(const ScoreMath& sm, f32x16_t& s) {
  if (sizeof(T) == 2 && sm.cap_out == 0.0f) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(s[i] * sm.cap_in));
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float x = s[i] * sm.cap_in;
      s[i] = sm.cap_out * (std::is_same<T, bf16>::value ? tanh_f32(x) : cap_tanh(x));
    }
  }
}

// The scores of keys that are not seen: the seen ones' bits first, then two operations a
// score on constants (compared one by one, the places held 30 registers through the loop).
template <typename T, int DB>
__device__ __forceinline__ void hide32(const Rows<T, DB>& r, f32x16_t& s, int key0, uint32_t seen) {
  const int half = (threadIdx.x & 63) >> 5;
  const auto below = [&](int key) { return (uint32_t)((1ull << max(0, min(key - key0, 32))) - 1); };
  const uint32_t bits = (seen & below(r.hi) & ~below(r.lo)) >> (4 * half);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint32_t keep = (uint32_t)((int32_t)(bits << (31 - (8 * (i / 4) + i % 4))) >> 31);
    s[i] = __uint_as_float((__float_as_uint(s[i]) & keep) | (0xff800000u & ~keep));
  }
}

// The weights are taken beside a reference m that follows the true maximum at a distance of
// up to 2^kLag: most units then leave what is summed up alone (raised at every new maximum,
// [4, 4096 ..] prompts took 709 us, with the lag 663). A row's largest weight is 2^kTop to
// 2^(kTop + kLag). bf16 and fp32 weights have the same digits at any size. fp16's end at 2^16,
// and below 2^-14 they lose digits, so they stand as high as they can, at 2^11 to 2^15: one
// keeps all of its digits down to 2^-25 of the row's largest, and is off by 2^-36 of it below
// (from 1 on, 8192 weights of 2^-25 each were left out of the products and counted in the sum).
//
// m is an exponent in base 2, c s - kTop, and a weight exp2(c s - m), one operation on the score.
// With c past 1 a finite score may leave fp32 there (bf16's lowest value times a scale of 1):
// then m is a score itself (its unit is c) and a weight exp2(c (s - m)).
template <typename T>
struct Reference {
  static constexpr bool kHalf = std::is_same<T, f16>::value;
  static constexpr float kLag = kHalf ? 4.0f : 8.0f, kTop = kHalf ? 11.0f : 0.0f;
  static constexpr bool kBare = !kHalf;  // (fp16's products end at 2^40)
  // What sums beside m are worth beside top (at least m).
  static __device__ __forceinline__ float factor(float m, float top, float unit2) {
    return top == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(kBare ? (m - top) * unit2 : m - top);
  }
};

template <typename T>
__device__ __forceinline__ ScoreMath score_math(Args g) {
  const bool bare = Reference<T>::kBare && g->unit2 != 1.0f;
  return {g->c, g->cap_in, g->cap_out, bare ? 1.0f : g->c, bare ? Reference<T>::kLag / g->unit2 : Reference<T>::kLag,
          g->cap_in > 0.0f, bare};
}

// Raises the references where N x 32 new scores ask for it, and makes the scores ready for
// weights32 (bare ones: less the reference).
template <typename T, int DB, int N>
__device__ __forceinline__ void new_maximum(const ScoreMath& sm, Rows<T, DB>& r, f32x16_t (&s)[N]) {
  using R = Reference<T>;
  float top = s[0][0];
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, s[n][i]);
  top = other_half_max(top);
  const float x = fmaf(top, sm.to_unit, -R::kTop);
  if (__any(x > r.m + sm.lag)) {
    const float m = fmaxf(r.m, x);
    const float keep = r.m == kNegInf ? 0.0f : R::factor(r.m, m, sm.bare ? sm.c : 1.0f);
    r.m = m;
    r.l *= keep;
#pragma unroll
    for (int b = 0; b < Shape<T, DB>::kBlocks; ++b) r.o[b] *= keep;
  }
  if (R::kBare && __builtin_expect(sm.bare, 0)) {
    const float m = r.m == kNegInf ? 0.0f : r.m;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[n][i] -= m;
  }
}

// The weights of 32 keys as the operand of their product: 16 bit rounded once, two to a
// register; fp32 as they are.
template <typename T>
struct Weights {
  u32x4 w[sizeof(T) == 2 ? 2 : 4];
};

template <typename T, int DB>
__device__ __forceinline__ Weights<T> weights32(const ScoreMath& sm, Rows<T, DB>& r, const f32x16_t& s) {
  // (nothing seen yet: every score is -inf or NaN, and the weight 0 or NaN)
  const float m = r.m == kNegInf || (Reference<T>::kBare && sm.bare) ? 0.0f : r.m;
  float p[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    p[i] = __builtin_amdgcn_exp2f(fmaf(s[i], sm.c, -m));
    r.l += p[i];
  }
  Weights<T> w;
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w.w[i / 4][i % 4] = pack2<T>(p[2 * i], p[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) w.w[i / 4][i % 4] = __float_as_uint(p[i]);
  }
  return w;
}

// O^T += V^T P^T of 32 keys.
template <typename T, int DB, int PITCH>
__device__ __forceinline__ void values32(Rows<T, DB>& r, const Weights<T>& p, const char* vl, int row0) {
  using S = Shape<T, DB>;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  if constexpr (sizeof(T) == 2) {
    // lane group q of 16 reads rows 4 (q / 2) + 0 .. 3 and 8 further on, columns 16 (q % 2) on
    const int j = lane & 15;
    const char* base = vl + (row0 + 4 * half + (j >> 2)) * PITCH + 32 * ((lane >> 4) & 1) + 8 * (j & 3);
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
      for (int blk = 0; blk < S::kBlocks; ++blk) {
        const u32x2 x = lds_tr(base + 16 * kb * PITCH + 64 * blk);
        const u32x2 y = lds_tr(base + (16 * kb + 8) * PITCH + 64 * blk);
        r.o[blk] = mfma32(T(), u32x4{x[0], x[1], y[0], y[1]}, p.w[kb], r.o[blk]);
      }
    }
  } else {
    const char* base = vl + (row0 + 4 * half) * PITCH + 4 * (lane & 31);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
#pragma unroll
      for (int blk = 0; blk < S::kBlocks; ++blk) {
        const float v = *reinterpret_cast<const float*>(base + (8 * (i / 4) + i % 4) * PITCH + 128 * blk);
        r.o[blk] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, __uint_as_float(p.w[i / 4][i % 4]), r.o[blk], 0, 0, 0);
      }
    }
  }
}

// The same for a unit of NB x 32 keys, for the matrix phase of the many-row kernel: the
// operands of a group of four MFMAs are read while the group before runs, and the compiler is
// kept from moving the reads back to their uses (it reads two operands, waits for them and
// uses them: [4, 4096 ..] prompts 531 us, left to the compiler 544).
__device__ __forceinline__ void pinned() { __builtin_amdgcn_sched_barrier(0); }

template <typename T, int DB, int NB>
__device__ __forceinline__ void scores_unit(const Rows<T, DB>& r, const char* kl, f32x16_t (&s)[NB]) {
  using S = Shape<T, DB>;
  constexpr int G = 4, kGroups = NB * S::kSteps / G;
  const int lane = threadIdx.x & 63;
  const char* base = kl + (lane & 31) * S::kPitch + 16 * (lane >> 5);
  u32x4 k[2][G];
  auto read = [&](int g) {
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const int at = g * G + i;
      k[g % 2][i] = *reinterpret_cast<const u32x4*>(base + (at / S::kSteps) * 32 * S::kPitch + 32 * (at % S::kSteps));
    }
  };
  read(0);
  pinned();
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    if (g + 1 < kGroups) read(g + 1);
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const int at = g * G + i, b = at / S::kSteps, step = at % S::kSteps;
      s[b] = mfma_step(T(), k[g % 2][i], r.q[step], step == 0 ? f32x16_t{} : s[b]);
    }
    pinned();
  }
}

template <typename T, int DB, int NB>
__device__ __forceinline__ void values_unit(Rows<T, DB>& r, const Weights<T> (&p)[NB], const char* vl) {
  using S = Shape<T, DB>;
  static_assert(sizeof(T) == 2, "fp32 takes values32");
  constexpr int G = S::kBlocks < 4 ? S::kBlocks : 4, kGroups = NB * 2 * S::kBlocks / G;
  const int lane = threadIdx.x & 63, j = lane & 15;
  const char* base = vl + (4 * (lane >> 5) + (j >> 2)) * S::vWidePitch + 32 * ((lane >> 4) & 1) + 8 * (j & 3);
  u32x2 x[2][G], y[2][G];
  auto read = [&](int g) {
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const int at = g * G + i;
      const char* from = base + 16 * (at / S::kBlocks) * S::vWidePitch + 64 * (at % S::kBlocks);
      x[g % 2][i] = lds_tr(from);
      y[g % 2][i] = lds_tr(from + 8 * S::vWidePitch);
    }
  };
  read(0);
  pinned();
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    if (g + 1 < kGroups) read(g + 1);
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const int at = g * G + i, kb = at / S::kBlocks, blk = at % S::kBlocks;
      const u32x2 a = x[g % 2][i], b = y[g % 2][i];
      r.o[blk] = mfma32(T(), u32x4{a[0], a[1], b[0], b[1]}, p[kb / 2].w[kb % 2], r.o[blk]);
    }
    pinned();
  }
}

// The lane's query's weight of key j of 32, as the product takes it.
template <typename T>
__device__ __forceinline__ float weight_at(const Weights<T>& p, int j) {
  const int lane = threadIdx.x & 63, i = 4 * (j >> 3) + (j & 3);  // its place in the half that has it
  constexpr int kEach = 4 / (int)sizeof(T), kWords = 16 / kEach;
  uint32_t x = 0;
#pragma unroll
  for (int k = 0; k < kWords; ++k) x = k == i / kEach ? p.w[k / 4][k % 4] : x;
  x = (uint32_t)__shfl((int)x, (lane & 31) + 32 * ((j >> 2) & 1));
  if constexpr (sizeof(T) == 4) return __uint_as_float(x);
  else return to_f32(__builtin_bit_cast(T, (uint16_t)(i & 1 ? x >> 16 : x)));
}

// Which of a lane's 16 weights are 0 as the product takes them: bits in their order (for the
// many-row kernel, which has no registers for the weights past their product).
template <typename T>
__device__ __forceinline__ uint32_t zero_weights(const Weights<T>& p) {
  constexpr int kEach = 4 / (int)sizeof(T);
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint32_t w = p.w[i / kEach / 4][i / kEach % 4], x = sizeof(T) == 4 ? w << 1 : (w >> (16 * (i % 2))) << 17;
    bits |= (x == 0 ? 1u : 0u) << i;
    asm volatile("" : "+v"(bits));  // one after the other: this path is rare, its registers are not
  }
  return bits;
}
// The weight of key j, or 1 for any that is not 0.
__device__ __forceinline__ float zero_or_one(uint32_t zero, int j) {
  const int lane = threadIdx.x & 63;
  const uint32_t its = (uint32_t)__shfl((int)zero, (lane & 31) + 32 * ((j >> 2) & 1));
  return (its >> (4 * (j >> 3) + (j & 3))) & 1 ? 0.0f : 1.0f;
}

// What values that are not finite (left out of LDS where only some rows see them) do to
// the rows that see their keys: times their weights (weight(j)), as in the product, they are
// themselves, or NaN beside a weight of 0.
template <typename T, int DB, typename W>
__device__ __forceinline__ void add_not_finite(Args g0, const Place& p, Rows<T, DB>& r, W weight, int key0, uint32_t seen) {
  const Args g = fresh(g0);
  const int half = (threadIdx.x & 63) >> 5, dim = g->a.dim;
  const PageMath math = page_math(g);
  const T* v0 = static_cast<const T*>(g->a.v) + (int64_t)p.h * g->a.vh;
  for (int j = 0; j < 32; ++j) {
    if (!((seen >> j) & 1)) continue;
    const int key = key0 + j;
    uint32_t i, slot;
    math.place((uint32_t)key, i, slot);
    const int64_t page = g->a.pages[(int64_t)p.b * g->a.ld_pages + i];  // (there: its bit is set)
    const T* v = v0 + page * g->a.vp + (int64_t)slot * g->a.vs;
    const bool sees = key < r.hi && key >= r.lo;
    const float w = weight(j);
#pragma unroll
    for (int blk = 0; blk < Shape<T, DB>::kBlocks; ++blk)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int d = 32 * blk + 8 * c + 4 * half;
        if (d < dim) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = to_f32(v[d + e]);
            if (sees && !(fabsf(x) < __builtin_inff())) r.o[blk][4 * c + e] += x * w;
          }
        }
        asm volatile("" ::: "memory");  // one load at a time: this path is rare, its registers are not
      }
  }
}

// Results of a wave's rows to the output.
template <typename T, int DB>
__device__ __forceinline__ void rows_out(Args g, int token, int head, int row, bool mine, const f32x16_t* o, float l) {
  const int half = (threadIdx.x & 63) >> 5;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int group = g->group, i = (uint32_t)row / (uint32_t)group, dim = g->a.dim;
  T* out = static_cast<T*>(g->a.out) + (int64_t)(token + i) * g->a.o_st + (int64_t)(head + (row - i * group)) * g->a.o_sh;
#pragma unroll
  for (int b = 0; b < Shape<T, DB>::kBlocks; ++b)
#pragma unroll
    for (int c = 0; c < 4; c += 2) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = o[b][4 * c + e] * inv;
      if constexpr (sizeof(T) == 2) {
        // the lane's 4 values of c and of c + 1 for 8 neighbours, with the other half's
        const auto lo = __builtin_amdgcn_permlane32_swap(pack2<T>(y[0], y[1]), pack2<T>(y[4], y[5]), false, false);
        const auto hi = __builtin_amdgcn_permlane32_swap(pack2<T>(y[2], y[3]), pack2<T>(y[6], y[7]), false, false);
        const int d = 32 * b + 8 * (c + half);
        if (mine && d < dim) *reinterpret_cast<u32x4*>(out + d) = u32x4{lo[0], hi[0], lo[1], hi[1]};
      } else {
        const int d = 32 * b + 8 * c + 4 * half;
        if (mine && d < dim) *reinterpret_cast<f32x4_v*>(out + d) = f32x4_v{y[0], y[1], y[2], y[3]};
        if (mine && d + 8 < dim) *reinterpret_cast<f32x4_v*>(out + d + 8) = f32x4_v{y[4], y[5], y[6], y[7]};
      }
    }
}

// A part of many rows holds its waves' registers as they are, four of a lane together: 1 KB
// a store (rows in order, as a part of few rows has them, took 14 us a tile of 256).
template <int DB>
__device__ __forceinline__ float* wave_part(Args g, int64_t slot, int wave) {
  return g->part + (slot * ((g->rows + 31) / 32) + wave) * (32 * (DB + 4));
}

// A row's results: to the output where the worker had all its units, else to a part's slot (-1: none).
template <typename T, int DB, bool MANY>
__device__ __forceinline__ void rows_end(Args g0, const Place& p, int row0, Rows<T, DB>& r, int64_t slot) {
  using S = Shape<T, DB>;
  const Args g = fresh(g0);
  const int lane = threadIdx.x & 63, half = lane >> 5, row = row0 + (lane & 31);
  const float l = both_halves(r.l);
  const int t0 = p.t * g->per_tile, tokens = min(g->per_tile, p.s.count - t0);
  const bool mine = row < tokens * g->group;
  if (slot < 0) {
    rows_out<T, DB>(g, p.s.first + t0, p.h * g->group, row, mine, r.o, l);
    return;
  }
  if (!mine) return;
  if constexpr (MANY) {
    float* x = wave_part<DB>(g, slot, row0 / kRows);
#pragma unroll
    for (int b = 0; b < S::kBlocks; ++b)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        *reinterpret_cast<f32x4_v*>(x + ((b * 4 + c) * 64 + lane) * 4) = f32x4_v{r.o[b][4 * c], r.o[b][4 * c + 1], r.o[b][4 * c + 2], r.o[b][4 * c + 3]};
    typedef float f32x2_v __attribute__((ext_vector_type(2)));
    *reinterpret_cast<f32x2_v*>(x + 32 * DB + 2 * lane) = f32x2_v{r.m, l};
  } else {
    float* x = g->part + (slot * g->rows + row) * (DB + 2);
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
  }
}

// The job that a worker leaves, given its last tile where it has begun that but not ended it.
__device__ __forceinline__ void leave_job(Args g0, int worker, const Place* p, int64_t slot, int parts) {
  const Args g = fresh(g0);
  Job j{};
  if (p != nullptr) {
    const int t0 = p->t * g->per_tile;
    j.first = slot;
    j.token = p->s.first + t0;
    j.head = p->h * g->group;
    j.rows = min(g->per_tile, p->s.count - t0) * g->group;
    j.parts = parts;
  }
  g->jobs[worker] = j;
}

// Zeros for the rows of no sequence, a token a wave at a time.
template <typename T>
__device__ __forceinline__ void zero_other_rows(Args g, int wave, int waves) {
  if (!g->a.zero_other || g->a.seq.starts == nullptr ||
      (g->a.seq.starts[0] <= 0 && g->a.seq.starts[g->a.seq.batch] >= g->a.seq.tokens))
    return;
  const Sequences s{g->a.seq.starts, g->a.seq.lengths, g->a.seq.batch, g->a.seq.tokens, g->a.seq.per};
  const int lane = threadIdx.x & 63;
  for (int64_t t = wave; t < s.tokens; t += waves) {
    if (sequence_of(s, (int)t) >= 0) continue;
    T* out = static_cast<T*>(g->a.out) + t * g->a.o_st;
    for (int h = 0; h < g->a.q_heads; ++h)
      for (int d = lane; d < g->a.dim; d += 64) out[h * g->a.o_sh + d] = from_f32<T>(0.0f);
  }
}

// Where the cache is: bases of this lane's chunk.
struct Cache {
  const char *k, *v;
  bool on;                 // the lane's chunk is one of a row
};

template <typename T, int DB>
__device__ __forceinline__ Cache cache_of(Args g) {
  using S = Shape<T, DB>;
  const int d = (threadIdx.x & 63) % S::kChunks * 16;
  return {static_cast<const char*>(g->a.k) + d, static_cast<const char*>(g->a.v) + d, d < g->a.dim * (int)sizeof(T)};
}

// Looking a key's row up, in two steps some units apart: its page is loaded (without a
// condition: a merge behind one would wait for it), then its K and V rows' byte offsets, or
// kNoRow, go into a table in LDS. The loops that read the table need nothing else of the
// sequence, head or page.
constexpr uint32_t kNoRow = 0xFFFFFFFFu;  // in the high half of K's offset

struct LookUp {
  int page, slot, h;
  bool of_tile;

  __device__ __forceinline__ void start(Args g0, const Place& p, int key) {
    const Args g = fresh(g0);
    of_tile = key >= p.k.lo && key < p.k.hi;
    uint32_t at, in;
    page_math(g).place((uint32_t)max(min(max(key, p.k.lo), p.k.hi - 1), 0), at, in);
    slot = (int)in;
    h = p.h;
    page = g->a.pages[(int64_t)p.b * g->a.ld_pages + at];
  }
  // Returns whether the key is there.
  template <typename T>
  __device__ __forceinline__ bool finish(Args g0, u32x4* to) const {
    const Args g = fresh(g0);
    const bool there = of_tile && (uint32_t)page < (uint32_t)g->a.n_pages;
    const uint64_t k = (uint64_t)(uint32_t)page * g->kp + (uint64_t)(uint32_t)slot * g->ks + (uint64_t)h * (uint64_t)(g->a.kh * (int64_t)sizeof(T));
    const uint64_t v = (uint64_t)(uint32_t)page * g->vp + (uint64_t)(uint32_t)slot * g->vs + (uint64_t)h * (uint64_t)(g->a.vh * (int64_t)sizeof(T));
    *to = u32x4{(uint32_t)k, there ? (uint32_t)(k >> 32) : kNoRow, (uint32_t)v, (uint32_t)(v >> 32)};
    return there;
  }
};

// Whether only some of a tile's rows see some of the unit's keys.
__device__ __forceinline__ bool partly_seen(Args g, const Place& p, int key0, int unit) {
  const int t0 = p.t * g->per_tile, tokens = min(g->per_tile, p.s.count - t0);
  bool some = tokens > 1 && key0 + unit > p.s.pos0 + t0 + 1;
  if (g->a.window > 0) some = some || (tokens > 1 && key0 < (int64_t)p.s.pos0 + t0 + tokens - g->a.window);
  return some;
}

// The K and V rows of a unit, as N loads of a wave each: load i takes rows first + i *
// stride .. + kPerLoad - 1. Rows that are not there are loaded from the cache's first place:
// their keys are hidden, their values become zeros on the way into LDS.
template <typename T, int DB, int N, int PITCH>
struct Loads {
  using S = Shape<T, DB>;
  u32x4 at[N];      // the rows' places, read from the table before they are needed
  u32x4 k[N], v[N];

  __device__ __forceinline__ void places(const u32x4* table, int first, int stride) {
    const int in = (threadIdx.x & 63) / S::kChunks;
#pragma unroll
    for (int i = 0; i < N; ++i) at[i] = table[first + i * stride + in];
  }

  // (lanes of chunks past the head's end load nothing: their part of LDS stays zeros)
  __device__ __forceinline__ void issue(const Cache& c) {
    if (!c.on) return;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bool row = at[i][1] != kNoRow;
      k[i] = *reinterpret_cast<const u32x4*>(c.k + (row ? (uint64_t)at[i][1] << 32 | at[i][0] : 0));
      v[i] = *reinterpret_cast<const u32x4*>(c.v + (row ? (uint64_t)at[i][3] << 32 | at[i][2] : 0));
    }
  }

  // Into LDS. gaps: not all rows of the unit are there (its table is given once more); clean:
  // values that are not finite become 0. Returns whether this lane had some of those.
  __device__ __forceinline__ bool store(const Cache& c, int first, int stride, char* kl, char* vl, bool gaps, const u32x4* table,
                                        bool clean) {
    if (!c.on) return false;
    const int lane = threadIdx.x & 63;
    const int row = first + lane / S::kChunks, chunk = lane % S::kChunks;
    char* kd = kl + row * S::kPitch + 16 * chunk;
    char* vd = vl + row * PITCH + 16 * chunk;
    uint32_t found = 0;
    if (gaps) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (table[row + i * stride][1] == kNoRow) v[i] = u32x4{0, 0, 0, 0};
    }
    if (clean) {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t bad = not_finite<T>(v[i][e]);
          found |= bad;
          v[i][e] = finite_only<T>(v[i][e], bad);
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      *reinterpret_cast<u32x4*>(kd + i * stride * S::kPitch) = k[i];
      *reinterpret_cast<u32x4*>(vd + i * stride * PITCH) = v[i];
    }
    return found != 0;
  }
};

// Zeros into LDS from all of a workgroup's (or wave's) threads.
__device__ __forceinline__ void clear_lds(char* to, int bytes, int thread, int threads) {
  for (int i = thread * 16; i < bytes; i += threads * 16) *reinterpret_cast<u32x4*>(to + i) = u32x4{0, 0, 0, 0};
}

// ---------------------------------------------------------------------------
// Few rows: a wave is a worker
// ---------------------------------------------------------------------------
// Bound by the cache's bytes, each read once: a wave loads a unit of 32 keys' K and V while
// it works on the one before, whose rows it has looked up a unit earlier. Of a tile of up to
// 32 rows the matrix cores do mostly nothing (a decode step has the group's heads), and are
// free. [64 sequences of 2048 to 8192 keys, 32 + 8 heads of 128] bf16 265 us, 5.1 TB/s, where
// reads alone reach 6.0; two of 130001 keys 180, 4.8 TB/s with the join. Rows of 512 bytes
// leave registers for one workgroup a CU, and still: 25 x 1882 keys, 4 heads of 256, bf16 51
// us, in tiles of many rows 70.
constexpr int kFewWaves = 4;

template <typename T, int DB>
__global__ void __launch_bounds__(64 * kFewWaves, DB * sizeof(T) <= 256 ? 2 : 1) attend_few_kernel(TileArgs, bool lined) {
  using S = Shape<T, DB>;
  constexpr int N = 32 / S::kPerLoad;
  __shared__ __attribute__((aligned(16))) char lds[kFewWaves][32 * (S::kPitch + S::vPitch)];
  __shared__ u32x4 tables[kFewWaves][2][64];  // the rows of two pairs of units
  __shared__ int64_t sums[kFewWaves];
  __shared__ int64_t found[kFewWaves][3];
  const Args g = kernel_args();
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int worker = blockIdx.x * kFewWaves + wave;
  const int batch = (int)g->a.seq.batch;
  int64_t total, n_workers, u0, u1, at = 0, units = 0;
  Place p;
  if (lined) {
    total = g->line[batch];
    n_workers = active_workers(g, total);
    u0 = begin_of(worker, total, n_workers);
    if (total > 0 && worker < n_workers) {
      p.b = sequence_at(g->line, batch, u0);
      at = g->line[p.b];
      units = g->line[p.b + 1] - at;
    }
  } else {
    // every workgroup lines the sequences up: 4 a thread, at most
    constexpr int kEach = kPlanBatch / (64 * kFewWaves);
    int64_t mine[kEach], sum = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int b = (int)threadIdx.x * kEach + i;
      mine[i] = b < batch ? units_of(g, seq_at(g, b), 0, 1) * g->a.kv_heads : 0;
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
    int64_t begins[kFewWaves];
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) begins[w] = begin_of((int64_t)blockIdx.x * kFewWaves + w, total, n_workers);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
#pragma unroll
      for (int w = 0; w < kFewWaves; ++w) {
        if (begins[w] >= before && begins[w] < before + mine[i]) {
          found[w][0] = (int)threadIdx.x * kEach + i;
          found[w][1] = before;
          found[w][2] = mine[i];
        }
      }
      before += mine[i];
    }
    __syncthreads();
    u0 = begin_of(worker, total, n_workers);
    p.b = uniform((int)found[wave][0]);
    at = found[wave][1];
    units = found[wave][2];
  }
  zero_other_rows<T>(g, worker, (int)gridDim.x * kFewWaves);
  if (total == 0 || worker >= n_workers) {
    if (lane == 0) leave_job(g, worker, nullptr, 0, 0);
    return;
  }
  u1 = begin_of(worker + 1, total, n_workers);
  int64_t in_tile = u0 - at;
  place_in_sequence(g, p, in_tile, units);

  char* const kl = lds[wave];
  char* const vl = lds[wave] + 32 * S::kPitch;
  const ScoreMath sm = score_math<T>(g);
  const Cache cache = cache_of<T, DB>(g);
  Loads<T, DB, N, S::vPitch> x;
  LookUp next;
  Rows<T, DB> r;
  if (g->a.dim < DB) clear_lds(kl, 32 * (S::kPitch + S::vPitch), lane, 64);
  int unit = uniform((int)in_tile), left = uniform((int)min(u1 - u0, (int64_t)INT32_MAX));
  for (int tile = 0;; ++tile) {
    const int begin = unit, tile_units = p.k.u1 - p.k.u0, n = min(tile_units - unit, left);
    int key = uniform((p.k.u0 + unit) * 32);
    // units are looked up in pairs: this one's are in the table, the next one's on their way
    next.start(g, p, key + lane);
    rows_load<T, DB>(g, p, 0, r);
    rows_begin<T, DB>(g, p, 0, r);
    uint64_t seen = __ballot(next.finish<T>(g, &tables[wave][0][lane]));
    next.start(g, p, key + 64 + lane);
    x.places(tables[wave][0], 0, S::kPerLoad);
    x.issue(cache);
    for (int i = 0; i < n; ++i, key += 32) {
      const uint32_t now = (uint32_t)seen;
      const bool mask = key < r.low || key + 32 > r.top || now != 0xFFFFFFFFu;
      const bool bad = x.store(cache, 0, S::kPerLoad, kl, vl, now != 0xFFFFFFFFu, &tables[wave][(i >> 1) & 1][(i & 1) * 32],
                               mask && (r.top < r.end || r.low > r.beg));
      seen >>= 32;
      if (i & 1) {
        seen = __ballot(next.finish<T>(g, &tables[wave][((i + 1) >> 1) & 1][lane]));
        next.start(g, p, key + 96 + lane);
      }
      if (i + 1 < n) {
        x.places(&tables[wave][((i + 1) >> 1) & 1][((i + 1) & 1) * 32], 0, S::kPerLoad);
        x.issue(cache);
      }
      f32x16_t s[1];
      s[0] = scores32<T, DB>(r, kl, 0);
      if (sm.cap) cap32<T>(sm, s[0]);
      if (mask) hide32<T, DB>(r, s[0], key, now);
      new_maximum<T, DB, 1>(sm, r, s);
      const Weights<T> w = weights32<T, DB>(sm, r, s[0]);
      values32<T, DB, S::vPitch>(r, w, vl, 0);
      if (__any(bad)) add_not_finite<T, DB>(g, p, r, [&](int j) { return weight_at<T>(w, j); }, key, now);
    }
    left -= n;
    unit += n;
    const bool ended = unit == tile_units;
    const int64_t slot = begin == 0 && ended ? -1 : 2 * (int64_t)worker + (tile > 0);
    rows_end<T, DB, false>(g, p, 0, r, slot);
    if (left == 0) {
      if (lane == 0) {
        const int parts = ended ? 0 : (int)(worker_of(u1 + (tile_units - unit) - 1, total, n_workers) - worker) + 1;
        leave_job(g, worker, begin == 0 && !ended ? &p : nullptr, slot, parts);
      }
      return;
    }
    unit = 0;
    next_place(g, p);
  }
}

// ---------------------------------------------------------------------------
// Many rows: a workgroup is a worker, its waves share the units' keys and values
// ---------------------------------------------------------------------------
// A worker's units go through a ring of LDS slots one after the other, whatever tile they
// are of. In a round of WAVES units each wave looks one of the next round's units up; a unit
// is loaded three and stored two steps before its scores are taken. A wave's step has two
// phases: the matrix cores' (O^T += of the unit before, the scores of this one; a tile's end
// and the next one's beginning between them; the stores and loads of units ahead) and the
// vector units' (the weights of this unit, look-ups). Half of the waves, one on each SIMD,
// runs a phase late, so that on every SIMD one wave feeds the matrix cores while the other
// computes weights. (Four waves of long rows have a SIMD each: all in one phase, and the
// stores after the barrier, which saves a slot.)
//
// Bound by what surrounds the products: prompts of up to 4096 tokens, 32 + 8 heads of 128 bf16,
// 485 to 505 us by card, 766 TFLOP/s where a product of 8192^3 reaches 1420. Of a step's 5600 cycles
// (1.9 GHz under this load) a SIMD's matrix cores take 2050. The matrix phase has 900 for O^T's
// products, 750 for the stores, loads and places of units ahead, 300 for tiles' ends, 660 for
// the scores, the vector phase 1340 for weights and 530 for look-ups. A first unit's operands
// read before the barrier, loads sent out in the vector phase, tiles of 64 rows a wave, two
// workgroups of four waves a CU: all the same or slower.
template <typename T, int DB, int WAVES, int UNIT>
__global__ void __launch_bounds__(64 * WAVES) attend_many_kernel(TileArgs, bool lined) {
  using S = Shape<T, DB>;
  constexpr int N = UNIT / S::kPerLoad / WAVES;  // loads of a wave, UNIT rows over all waves
  constexpr int NB = UNIT / 32;
  static_assert(N >= 1 && N * S::kPerLoad * WAVES == UNIT, "a unit is whole loads of every wave");
  // Units that are stored before they are used (one where the rows are too long for more);
  // K is read in the step of its scores, V in the next one, by the late waves a phase later.
  constexpr int kAhead = S::kRowBytes > 512 ? 1 : 2;
  constexpr int kSlots = kAhead + (WAVES == 8), vSlots = kSlots + 1;
  // The rows' table holds 16 units: the rounds that are used and kLead more.
  constexpr int kTable = 16, kLead = WAVES == 8 ? 1 : 2, kFinish = 2;
  static_assert(WAVES == 8 || WAVES == 4, "rounds divide the table");
  __shared__ __attribute__((aligned(16))) char kl[kSlots][UNIT * S::kPitch];
  __shared__ __attribute__((aligned(16))) char vl[vSlots][UNIT * S::vWidePitch];
  __shared__ u32x4 table[kTable][UNIT];
  __shared__ uint32_t there[2 * kTable][4];      // of a unit: the bits of its keys that are there; 1: partly seen, 2: not all there
  __shared__ int64_t own_line[kPlanMany + 1];    // the line of a call of few sequences
  __shared__ int bad[vSlots];                    // the unit (by count) whose values are not all finite
  const Args g = kernel_args();
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const bool late = WAVES == 8 && wave >= 4;
  // neighbours in the line, which share keys, go to one XCD
  const int nb = (int)gridDim.x;
  const int worker = nb % 8 == 0 ? (int)(blockIdx.x % 8) * (nb / 8) + (int)blockIdx.x / 8 : (int)blockIdx.x;
  const int batch = (int)g->a.seq.batch;
  if (!lined) {
    for (int b = wave; b < batch; b += WAVES) {
      const int64_t n = wave_sum64(units_of(g, seq_at(g, b), lane, 64));
      if (lane == 0) own_line[b + 1] = n * g->a.kv_heads;
    }
    __syncthreads();
    if (wave == 0) {
      int64_t upto = lane < batch ? own_line[lane + 1] : 0;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int64_t o = __shfl_up(upto, d);
        if (lane >= d) upto += o;
      }
      if (lane == 0) own_line[0] = 0;
      own_line[lane + 1] = upto;
    }
    __syncthreads();
  }
  const int64_t total = uniform64(lined ? g->line[batch] : own_line[batch]);
  const int64_t n_workers = active_workers(g, total);
  zero_other_rows<T>(g, worker * WAVES + wave, nb * WAVES);
  if (total == 0 || worker >= n_workers) {
    if (threadIdx.x == 0) leave_job(g, worker, nullptr, 0, 0);
    return;
  }
  const int64_t u0 = begin_of(worker, total, n_workers), u1 = begin_of(worker + 1, total, n_workers);
  const int n = uniform((int)min(u1 - u0, (int64_t)INT32_MAX));
  Place p;
  p.b = lined ? sequence_at(g->line, batch, u0) : sequence_at(own_line, batch, u0);
  const int64_t at = uniform64(lined ? g->line[p.b] : own_line[p.b]);
  const int64_t next_at = uniform64(lined ? g->line[p.b + 1] : own_line[p.b + 1]);
  int64_t in_tile = u0 - at;
  place_in_sequence(g, p, in_tile, next_at - at);
  const int row0 = wave * kRows, first = wave * S::kPerLoad;
  constexpr int stride = WAVES * S::kPerLoad;
  const ScoreMath sm = score_math<T>(g);
  const Cache cache = cache_of<T, DB>(g);

  // this wave's units on their way: the one that it looks up next
  LookUp next;
  Place lp = p;
  int l_unit = uniform((int)in_tile), l_at = 0;
  auto advance = [&](int by) {
    l_at += by;
    if (l_unit + by < lp.k.u1 - lp.k.u0) {
      l_unit += by;
      return;
    }
    while (by > 0 && l_at < n) {
      const int rest = lp.k.u1 - lp.k.u0 - l_unit, go = min(by, rest);
      l_unit += go;
      by -= go;
      if (go == rest) {
        l_unit = 0;
        next_place(fresh(g), lp);
      }
    }
  };
  auto start = [&]() {
    if (l_at < n) next.start(g, lp, (lp.k.u0 + l_unit) * UNIT + (lane & (UNIT - 1)));
  };
  auto finish = [&]() {
    if (l_at < n) {
      const int at = l_at % (2 * kTable);
      const bool key_there = lane < UNIT && next.finish<T>(g, &table[at % kTable][lane & (UNIT - 1)]);
      const uint64_t bits = __ballot(key_there);
      const bool some = partly_seen(fresh(g), lp, (lp.k.u0 + l_unit) * UNIT, UNIT);
      if (lane == 0) {
        there[at][0] = (uint32_t)bits;
        there[at][1] = (uint32_t)(bits >> 32);
        there[at][2] = some | (bits != (UNIT == 64 ? ~0ull : 0xFFFFFFFFull)) * 2u;
      }
      advance(WAVES);
    }
  };
  auto seen_of = [&](int j) {
    const uint32_t* t = there[j % (2 * kTable)];
    return (uint64_t)(uint32_t)uniform(t[1]) << 32 | (uint32_t)uniform(t[0]);
  };
  Loads<T, DB, N, S::vWidePitch> x;
  int kput = 0, vput = 0;  // the slots that are stored next
  uint32_t flags = 0;      // of the unit that is stored next
  auto prepare = [&](int j) {
    x.places(table[j % kTable], first, stride);
    flags = there[(j + 2 * kTable - 1) % (2 * kTable)][2];
  };
  // Unit j into LDS, the next one on its way, the one after it made ready: nothing here waits
  // for what it has asked for itself.
  auto bring = [&](int j) {
    if (j >= n) return;
    const int f = uniform(flags);
    if (x.store(cache, first, stride, kl[kput], vl[vput], f & 2, table[j % kTable], f & 1)) bad[vput] = j + 1;
    kput = kput + 1 == kSlots ? 0 : kput + 1;
    vput = vput + 1 == vSlots ? 0 : vput + 1;
    if (j + 1 < n) {
      x.issue(cache);
      prepare(j + 2);
    }
  };
  if (threadIdx.x < vSlots) bad[threadIdx.x] = 0;
  if (g->a.dim < DB) {
    clear_lds(kl[0], sizeof(kl), threadIdx.x, 64 * WAVES);
    clear_lds(vl[0], sizeof(vl), threadIdx.x, 64 * WAVES);
  }
  advance(wave);
  for (int a = 0; a < kLead; ++a) {
    start();
    finish();
  }
  Rows<T, DB> r;
  rows_load<T, DB>(g, p, row0, r);
  rows_begin<T, DB>(g, p, row0, r);
  __syncthreads();
  prepare(0);
  x.issue(cache);
  prepare(1);
  for (int a = 0; a < kAhead; ++a) bring(a);
  __syncthreads();
  if (late) __syncthreads();

  int kget = 0, vget = vSlots - 1;  // the slots of unit j's keys and of unit j - 1's values
  bool before = false;              // this wave has weights of unit j - 1
  int unit = uniform((int)in_tile), begin = unit, tiles = 0;  // of the tile: unit j, this worker's first
  int key = uniform((p.k.u0 + unit) * UNIT), units = uniform(p.k.u1 - p.k.u0);
  Place following = p;
  Weights<T> w[NB];
  int spoilt = 0;                   // unit j - 1 has values that are not finite where it is j
  for (int j = 0;; ++j) {
    __builtin_amdgcn_s_setprio(1);  // the matrix cores' wave first
    if (before) {
      uint32_t zero = 0;
      if (__builtin_expect(spoilt == j, 0)) {
#pragma unroll
        for (int b = 0; b < NB; ++b) zero |= zero_weights<T>(w[b]) << (16 * b);
      }
      if constexpr (sizeof(T) == 2) {
        values_unit<T, DB, NB>(r, w, vl[vget]);
      } else {
#pragma unroll
        for (int b = 0; b < NB; ++b) values32<T, DB, S::vWidePitch>(r, w[b], vl[vget], 32 * b);
      }
      if (__builtin_expect(spoilt == j, 0)) {
        const uint64_t seen = seen_of(j - 1);
        for (int b = 0; b < NB; ++b)
          add_not_finite<T, DB>(g, p, r, [&](int j) { return zero_or_one(zero >> (16 * b), j); }, key - UNIT + 32 * b,
                                (uint32_t)(seen >> (32 * b)));
      }
    }
    // Queries that may be on their way are waited for here, where the unit's loads are, too:
    // before the scores the wait would include the loads that `bring` has just sent out.
#pragma unroll
    for (int k = 0; k < S::kSteps; ++k) asm volatile("" : "+v"(r.q[k]));
    // (ahead of a tile's stores, whose end the wait for the loads would include)
    if (WAVES == 8) bring(j + kAhead);
    const bool ended = j > 0 && unit == units;
    if (ended || j == n) {
      const int64_t slot = begin == 0 && ended ? -1 : 2 * (int64_t)worker + (tiles > 0);
      rows_end<T, DB, true>(g, p, row0, r, slot);
      if (j == n) {
        if (threadIdx.x == 0) {
          const int last = (int)fresh(g)->a.seq.batch;
          const int64_t all = lined ? fresh(g)->line[last] : own_line[last], count = active_workers(fresh(g), all);
          const int64_t end = begin_of(worker + 1, all, count);
          const int parts = ended ? 0 : (int)(worker_of(end + (units - unit) - 1, all, count) - worker) + 1;
          leave_job(g, worker, begin == 0 && !ended ? &p : nullptr, slot, parts);
        }
        break;
      }
      p = following;
      unit = begin = 0;
      ++tiles;
      key = uniform(p.k.u0 * UNIT);
      units = uniform(p.k.u1 - p.k.u0);
      rows_begin<T, DB>(g, p, row0, r);
    }
    const bool now = key < r.end && key + UNIT > r.beg;
    f32x16_t s[NB];  // (of this step alone: set where it is read, in no other registers)
    if (now) scores_unit<T, DB, NB>(r, kl[kget], s);
    __builtin_amdgcn_s_setprio(0);
    __syncthreads();
    if (WAVES != 8) bring(j + kAhead);
    if (unit + 1 == units && j + 1 < n) {  // the next tile's queries, in the registers that the last scores have left
      following = p;
      next_place(fresh(g), following);
      rows_load<T, DB>(g, following, row0, r);
    }
    if (j % WAVES == 0) start();
    if (j % WAVES == kFinish) finish();
    if (now) {
      if (sm.cap) {
#pragma unroll
        for (int b = 0; b < NB; ++b) cap32<T>(sm, s[b]);
      }
      const uint64_t seen = seen_of(j);
      const int spoilt_by = bad[vget + 1 == vSlots ? 0 : vget + 1];
      if (key < r.low || key + UNIT > r.top || seen != (UNIT == 64 ? ~0ull : 0xFFFFFFFFull)) {
#pragma unroll
        for (int b = 0; b < NB; ++b) hide32<T, DB>(r, s[b], key + 32 * b, (uint32_t)(seen >> (32 * b)));
      }
      new_maximum<T, DB, NB>(sm, r, s);
#pragma unroll
      for (int b = 0; b < NB; ++b) w[b] = weights32<T, DB>(sm, r, s[b]);
      spoilt = uniform(spoilt_by);
    }
    before = now;
    ++unit;
    key += UNIT;
    kget = kget + 1 == kSlots ? 0 : kget + 1;
    vget = vget + 1 == vSlots ? 0 : vget + 1;
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Joining the parts: a job for each worker whose last tile goes on in the next one
// ---------------------------------------------------------------------------
// Of many rows: a workgroup for 32 of them, the parts over its waves, then wave 0 takes the
// others' sums in their order.
template <typename T, int DB>
__global__ void __launch_bounds__(256) attend_join_many_kernel(TileArgs) {
  typedef float f32x2_v __attribute__((ext_vector_type(2)));
  __shared__ f32x4_v sums[3][DB / 8][64];
  __shared__ f32x2_v stats[3][64];
  const Args g = kernel_args();
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), block = blockIdx.y;
  const Job job = g->jobs[blockIdx.x];
  const int row = block * kRows + (lane & 31);
  if (block * kRows >= job.rows) return;
  const bool mine = row < job.rows;
  f32x16_t o[DB / 32];
#pragma unroll
  for (int b = 0; b < DB / 32; ++b) o[b] = f32x16_t{};
  const float unit2 = g->unit2;
  float top = kNegInf, sum = 0.0f;
  // adds (ml, what `from` gives) to the sums
  const auto add = [&](f32x2_v ml, auto from) {
    const float now = fmaxf(top, ml[0]), keep = Reference<T>::factor(top, now, unit2), f = Reference<T>::factor(ml[0], now, unit2);
    top = now;
    sum = sum * keep + ml[1] * f;
#pragma unroll
    for (int b = 0; b < DB / 32; ++b)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const f32x4_v v = from(b * 4 + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[b][4 * c + e] = o[b][4 * c + e] * keep + v[e] * f;
      }
  };
  for (int i = wave; i < job.parts; i += 4) {
    const float* x = wave_part<DB>(g, i == 0 ? job.first : 2 * ((int64_t)blockIdx.x + i), block);
    f32x2_v ml = {kNegInf, 0.0f};  // (lanes without a row left nothing)
    if (mine) ml = *reinterpret_cast<const f32x2_v*>(x + 32 * DB + 2 * lane);
    add(ml, [&](int at) {
      f32x4_v v = {0.0f, 0.0f, 0.0f, 0.0f};
      if (mine) v = *reinterpret_cast<const f32x4_v*>(x + (at * 64 + lane) * 4);
      return v;
    });
  }
  if (wave > 0) {
    stats[wave - 1][lane] = f32x2_v{top, sum};
#pragma unroll
    for (int at = 0; at < DB / 8; ++at)
      sums[wave - 1][at][lane] = f32x4_v{o[at / 4][4 * (at % 4)], o[at / 4][4 * (at % 4) + 1], o[at / 4][4 * (at % 4) + 2], o[at / 4][4 * (at % 4) + 3]};
  }
  __syncthreads();
  if (wave > 0) return;
  for (int w = 0; w < min(job.parts - 1, 3); ++w) add(stats[w][lane], [&](int at) { return sums[w][at][lane]; });
  rows_out<T, DB>(g, job.token, job.head, row, mine, o, sum);
}

template <typename T, int DB>
__global__ void __launch_bounds__(256) attend_join_kernel(TileArgs) {
  constexpr int kVals = DB / 64;
  const Args g = kernel_args();
  __shared__ float sums[4][DB];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Job job = g->jobs[blockIdx.x];
  const int rows = job.rows, parts = job.parts;
  if (rows == 0) return;
  const int64_t one = (int64_t)g->rows * (DB + 2);
  const float* first = g->part + job.first * one;
  const float* rest = g->part + 2 * ((int64_t)blockIdx.x + 1) * one;  // part i > 0: two slots further each
  auto part = [&](int i, int row) { return (i == 0 ? first : rest + (int64_t)(i - 1) * 2 * one) + (int64_t)row * (DB + 2); };
  auto store = [&](int row, const float* acc, float inv) {
    const int i = (uint32_t)row / (uint32_t)g->group;
    T* out = static_cast<T*>(g->a.out) + (int64_t)(job.token + i) * g->a.o_st + (int64_t)(job.head + row - i * g->group) * g->a.o_sh;
#pragma unroll
    for (int v = 0; v < kVals; ++v)
      if (64 * v + lane < g->a.dim) out[64 * v + lane] = from_f32<T>(acc[v] * inv);
  };
  typedef float f32x2_a __attribute__((ext_vector_type(2), aligned(8)));
  const float unit2 = g->unit2;
  const auto factor = [&](float m, float top) { return Reference<T>::factor(m, top, unit2); };
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
  float join_cost;
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
  p.few = max_chunk * group <= kRows && p.padded * (f32 ? 4 : 2) <= 512;
  p.waves = p.few || wide ? 4 : 8;
  p.unit = p.few || wide ? 32 : 64;
  const int64_t rows = p.few ? kRows : kRows * p.waves;
  p.per_tile = (int)std::max((int64_t)1, std::min(rows / group, max_chunk));
  p.rows = (int)(p.per_tile * group);
  // least units of a worker: of one token over 777 keys 1: 14.2 us, 2: 16.8, 4: 18.5, 32: 43.6
  // (of many rows 1 to 8 are alike)
  p.min_units = p.few ? 1 : 2;
  // (a thread of the few-row kernel lines up a whole sequence: of many tiles, by an understated
  // max_chunk, 64 lanes do)
  p.lined = batch > (p.few ? kPlanBatch : kPlanMany) || (p.few && tokens / p.per_tile > batch + 4096);
  // workgroups at once: two of the few-row kernel where their LDS and registers leave room
  const int64_t groups = (int64_t)cu_count() * (p.few && !wide ? 2 : 1);
  const double most = (double)kv_heads * ((double)tokens / p.per_tile + (double)batch) * ((double)max_keys / p.unit + 1.0);
  const int64_t useful = most > 1e9 ? (int64_t)1 << 30 : (int64_t)most / p.min_units + 1;
  p.workers = std::min(groups * (p.few ? kFewWaves : 1), useful);
  if (p.few) p.workers = (p.workers + kFewWaves - 1) / kFewWaves * kFewWaves;
  const int64_t tiles = kv_heads * std::max(tokens / p.per_tile, (int64_t)1);
  p.cut = p.workers > 8 * tiles;
  // (measured: half and double of either cost do the same on the average of random calls. Units of
  // fp32 take four times as long: with that in the cost chunks of 11 tokens over 3 x 2654 keys, 4
  // heads of 96, take 44 us, without it 47; ten other random calls of fp32 the same either way)
  p.join_cost = (p.few ? 0.02f * (float)((p.rows + 15) / 16) : 0.2f) / (f32 ? 4.0f : 1.0f) / (float)tiles;
  p.line_bytes = (size_t)(batch + 2) / 2 * 16;
  p.job_bytes = ((size_t)p.workers * sizeof(Job) + 15) / 16 * 16;  // (the parts behind them are read 16 bytes at a time)
  const size_t part = p.few ? (size_t)p.rows * (size_t)(p.padded + 2) : (size_t)((p.rows + 31) / 32) * 32 * (size_t)(p.padded + 4);
  p.part_bytes = (size_t)p.workers * 2 * part * sizeof(float);
  return p;
}

template <typename T, int DB>
void launch_tiles(const TileArgs& g, const Plan& p, hipStream_t s) {
  if (p.lined) attend_line_kernel<<<dim3(1), dim3(1024), 0, s>>>(g);
  if constexpr (DB * sizeof(T) <= 512) {
    if (p.few) attend_few_kernel<T, DB><<<dim3((unsigned)(p.workers / kFewWaves)), dim3(64 * kFewWaves), 0, s>>>(g, p.lined);
  }
  if (!p.few) {
    constexpr int kWaves = DB * sizeof(T) > 256 ? 4 : 8, kUnit = DB * sizeof(T) > 256 ? 32 : 64;
    attend_many_kernel<T, DB, kWaves, kUnit><<<dim3((unsigned)p.workers), dim3(64 * kWaves), 0, s>>>(g, p.lined);
  }
  if (p.workers > 1) {
    const unsigned jobs = (unsigned)(p.workers - 1);
    if (!p.few) attend_join_many_kernel<T, DB><<<dim3(jobs, (unsigned)((p.rows + 31) / 32)), dim3(256), 0, s>>>(g);
    // (of few rows in many parts a row a workgroup, up to 16: with 4 the two calls above took 59 and 50 us)
    else attend_join_kernel<T, DB><<<dim3(jobs, (unsigned)(p.cut ? std::min(p.rows, 16) : 1)), dim3(256), 0, s>>>(g);
  }
}

template <typename T>
void launch_type(TileArgs& g, const Plan& p, hipStream_t s) {
  auto go = [&](auto db) { launch_tiles<T, decltype(db)::value>(g, p, s); };
  if (p.padded == 64) go(std::integral_constant<int, 64>());
  else if (p.padded == 128) go(std::integral_constant<int, 128>());
  else go(std::integral_constant<int, 256>());
}

}  // namespace

bool attend_tiles_take(const AttendArgs& a, int dtype) {
  const int ve = 16 / ak_dtype_size(dtype);
  const int64_t group = a.q_heads / a.kv_heads;
  bool ok = a.max_pages > 0 && a.n_pages > 0 && a.dim <= 256 && a.dim % ve == 0 && group <= kRows * (a.dim > 128 || (a.dim > 64 && ve == 4) ? 4 : 8);
  for (const void* x : {a.q, a.k, a.v, (const void*)a.out}) ok = ok && aligned16(x);
  for (int64_t st : {a.q_st, a.q_sh, a.o_st, a.o_sh, a.kp, a.ks, a.kh, a.vp, a.vs, a.vh}) ok = ok && st % ve == 0;
  for (int64_t st : {a.kp, a.ks, a.vp, a.vs}) ok = ok && st <= (int64_t)UINT32_MAX / 4;  // (bytes are multiplied in 32 x 32 bits)
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
  g.join_cost = p.join_cost;
  const uint32_t esz = (uint32_t)ak_dtype_size(dtype);
  g.kp = (uint32_t)a.kp * esz;
  g.ks = (uint32_t)a.ks * esz;
  g.vp = (uint32_t)a.vp * esz;
  g.vs = (uint32_t)a.vs * esz;
  g.line = static_cast<int64_t*>(workspace);
  g.jobs = reinterpret_cast<Job*>(static_cast<char*>(workspace) + p.line_bytes);
  g.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.line_bytes + p.job_bytes);
  if (a.softcap > 0.0f && a.softcap <= kQuickCap && esz == 2) {
    g.cap_in = 2.0f * kLog2e * (a.scale / a.softcap);
    g.c = 2.0f * kLog2e * a.softcap;
  } else if (a.softcap > 0.0f) {
    g.cap_in = a.scale / a.softcap;
    g.cap_out = a.softcap * kLog2e;
    g.c = 1.0f;
  } else {
    g.c = a.scale * kLog2e;
  }
  // (capped scores stay below 2^15 in base 2)
  g.unit2 = a.softcap == 0.0f && g.c > 1.0f && dtype != AK_DTYPE_F16 ? g.c : 1.0f;
  if (dtype == AK_DTYPE_F32) launch_type<float>(g, p, s);
  else if (dtype == AK_DTYPE_F16) launch_type<f16>(g, p, s);
  else launch_type<bf16>(g, p, s);
}

}  // namespace ak
