// Rotary positions, head norms and the paged cache's appends for gfx950.
//
// Per token and head of dim elements, in fp32 with one final rounding:
//   n = x / sqrt(mean(x^2) + eps) * weight     (where the heads are normed)
//   y = the pairs of n's first `rotary` elements turned by the token's angles,
//       (y0, y1) = (n0 cos - n1 sin, n1 cos + n0 sin), the rest as it is
// A pair is (i, i + rotary / 2), or interleaved (2 i, 2 i + 1). The cosines and
// sines of a position are a row of an fp32 table ([positions][2][rotary / 2],
// made once in float64): an angle of a far position in fp32 has lost the digits
// that matter. Backward, with dz = dy turned back and r = 1 / rms:
//   dx = r (g - n mean(g n)),  g = dz weight,  n = x r;  dweight = sum of dz n
//
// HBM-bound: every element is read once and written once, the table's rows
// come from the caches. One head's row belongs to the fewest lanes (a power of
// two) that hold it in units of two 16-byte vectors: the two vectors of a unit
// hold the two halves of its pairs, so the turn needs no exchange between
// lanes, and only the norm's sum crosses them (DPP).
#include <algorithm>
#include <utility>

#include "heads.h"

namespace ak {
namespace {

constexpr int kThreads = 256;
// Results that the eight L2s of 4 MiB cannot hold are stored past them: 84 MB of
// queries and keys turned there and back in 65 us (5.2 TB/s; on other cards up to 70),
// through them in 79 (normed too, in 85 to 90 and 93). Smaller ones stay for their
// reader; so does what goes into a cache, 67 us for 133 MB of appended prompts, past
// the L2s 66.
constexpr int64_t kL2Bytes = 32 << 20;

// One of the tensors whose heads a call walks over: element strides, the last
// dimension dense.
struct HeadRows {
  const void* x;
  void* y;
  const void* w;      // the norm's weight, or NULL
  int64_t so, si, sh; // of x: outer, inner (token), head
  int64_t yt, ys, yh; // of y: token and head; of a cache: page, slot and head
  int64_t heads;
};

struct HeadArgs {
  HeadRows r[3];      // queries, keys, values (the last two into the cache where there is one)
  const float* table;
  const void* positions;
  int64_t tokens, inner, n_positions, table_rows;
  int64_t all_heads, total;  // heads of all tensors, rows: tokens times them
  Divisor by_heads, by_inner, by_positions, by_page;  // for whole vectors' rows, where all numbers have 32 bits
  int dim, rotary, lpr_log2;
  int interleaved, inverse, pos64, zero_tail;
  int past;           // results go past the L2s
  float eps, by_dim;  // by_dim: 1 / dim
  // the cache
  Sequences seq;
  const int32_t* pages;
  int64_t n_pages, page_size, max_pages, ld_pages;
};

// Rows are counted in 64 bits, or where the numbers allow it in 32: in 64 their places
// took more than half of the instructions (appended prompts 67 us, in 32 53).
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b, const Divisor&) {
  if (((a | b) >> 32) == 0) return (uint32_t)a / (uint32_t)b;
  return a / b;
}
__device__ __forceinline__ uint32_t quotient(uint32_t a, int64_t, const Divisor& by) { return by(a); }
__device__ __forceinline__ int64_t steps(int64_t n, int64_t stride) { return n * stride; }
__device__ __forceinline__ int64_t steps(uint32_t n, int64_t stride) { return (int64_t)((uint64_t)n * (uint32_t)stride); }

// N elements in one access of 16, 8 or 4 bytes.
template <int BYTES>
struct Word;
template <>
struct Word<16> { typedef u32x4 type; };
template <>
struct Word<8> { typedef uint32_t type __attribute__((ext_vector_type(2))); };
template <>
struct Word<4> { typedef uint32_t type; };

template <typename T, int N>
union Vec {
  typedef typename Word<N * sizeof(T)>::type W;
  W u;
  T e[N];
};

template <int N, typename T>
__device__ __forceinline__ Vec<T, N> load_vec(const T* p) {
  Vec<T, N> v;
  v.u = *reinterpret_cast<const typename Vec<T, N>::W*>(p);
  return v;
}

template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, N>& v) {
  *reinterpret_cast<typename Vec<T, N>::W*>(p) = v.u;
}
template <typename T, int N>
__device__ __forceinline__ void store_past(T* p, const Vec<T, N>& v) {
  __builtin_nontemporal_store(v.u, reinterpret_cast<typename Vec<T, N>::W*>(p));
}

// The sum over the 2^log2 lanes of a row (aligned to their number).
__device__ __forceinline__ float lanes_sum(float v, int log2) {
  if (log2 > 0) v += dpp<kDppXor1>(v);
  if (log2 > 1) v += dpp<kDppXor2>(v);
  if (log2 > 2) v += dpp<kDppHalfMirror>(v);
  if (log2 > 3) v += dpp<kDppMirror>(v);
  if (log2 > 4) v += __shfl_xor(v, 16, kWave);
  if (log2 > 5) v += __shfl_xor(v, 32, kWave);
  return v;
}

// Where a unit's two vectors stand in the head, and whether they are turned.
template <int VE>
struct Unit {
  int off0, off1;
  bool turned, has0, has1;
  __device__ __forceinline__ Unit(int u, const HeadArgs& a) {
    const int ur = a.rotary / (2 * VE);
    turned = u < ur;
    const bool halves = turned & !a.interleaved;  // else its two vectors are neighbours
    off0 = halves ? u * VE : 2 * u * VE;
    off1 = off0 + (halves ? a.rotary / 2 : VE);
    has0 = off0 < a.dim;
    has1 = off1 < a.dim;
  }
};

// The angles of a unit's VE pairs: cosines and sines (negated for the way back).
template <int VE, bool INVERSE>
__device__ __forceinline__ void load_angles(const HeadArgs& a, int64_t pos, int u, float (&c)[VE], float (&s)[VE]) {
  constexpr int A = VE < 4 ? VE : 4;
  Vec<float, A> cv[VE / A], sv[VE / A];
#pragma unroll
  for (int e = 0; e < VE; ++e) cv[e / A].e[e % A] = sv[e / A].e[e % A] = __builtin_nanf("");
  if (pos >= 0 && pos < a.table_rows) {
    const float* row = a.table + steps((uint32_t)pos, a.rotary) + u * VE;
#pragma unroll
    for (int i = 0; i < VE / A; ++i) {
      cv[i] = load_vec<A>(row + A * i);
      sv[i] = load_vec<A>(row + a.rotary / 2 + A * i);
    }
  }
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    c[e] = cv[e / A].e[e % A];
    s[e] = INVERSE && a.inverse ? -sv[e / A].e[e % A] : sv[e / A].e[e % A];
  }
}

template <int VE>
__device__ __forceinline__ void turn(float (&p)[VE], float (&q)[VE], const float (&c)[VE], const float (&s)[VE],
                                     bool interleaved) {
  if (interleaved) {
#pragma unroll
    for (int e = 0; e < VE; e += 2) {
      const float p0 = p[e], p1 = p[e + 1], q0 = q[e], q1 = q[e + 1];
      const float pc = c[e / 2], ps = s[e / 2], qc = c[VE / 2 + e / 2], qs = s[VE / 2 + e / 2];
      p[e] = p0 * pc - p1 * ps;
      p[e + 1] = p1 * pc + p0 * ps;
      q[e] = q0 * qc - q1 * qs;
      q[e + 1] = q1 * qc + q0 * qs;
    }
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const float x0 = p[e], x1 = q[e];
      p[e] = x0 * c[e] - x1 * s[e];
      q[e] = x1 * c[e] + x0 * s[e];
    }
  }
}

template <typename I>
__device__ __forceinline__ int64_t position_of(const HeadArgs& a, I token) {
  const I n = (I)a.n_positions, i = token < n ? token : token - quotient(token, a.n_positions, a.by_positions) * n;
  if (a.positions == nullptr) return i;
  return a.pos64 ? static_cast<const int64_t*>(a.positions)[i] : (int64_t)static_cast<const int32_t*>(a.positions)[i];
}

// What a row of the walk is: its tensor, token and head, and where it is read.
template <typename T, typename I>
struct Row {
  const T* x;
  const T* w;
  I token, h;
  int kind;
};

// (field by field: an index would put the arguments into scratch memory)
#define AK_PICK(f) (kind == 0 ? a.r[0].f : kind == 1 ? a.r[1].f : a.r[2].f)

template <typename T, bool APPEND, typename I>
__device__ __forceinline__ Row<T, I> row_of(const HeadArgs& a, I row) {
  Row<T, I> o;
  o.token = quotient(row, a.all_heads, a.by_heads);
  I h = row - o.token * (I)a.all_heads;
  int kind = 0;
  if (h >= (I)a.r[0].heads) {
    h -= (I)a.r[0].heads;
    kind = 1;
    if (APPEND && h >= (I)a.r[1].heads) {
      h -= (I)a.r[1].heads;
      kind = 2;
    }
  }
  o.h = h;
  o.kind = kind;
  o.x = static_cast<const T*>(AK_PICK(x)) + steps(h, AK_PICK(sh));
  if (!APPEND && a.inner < a.tokens) {
    const I outer = quotient(o.token, a.inner, a.by_inner);
    o.x += steps(outer, AK_PICK(so)) + steps(o.token - outer * (I)a.inner, AK_PICK(si));
  } else {
    o.x += steps(o.token, AK_PICK(si));
  }
  o.w = static_cast<const T*>(AK_PICK(w));
  return o;
}

// Where it is written, and the position whose angles turn it.
template <typename T>
struct Target {
  T* y;
  int64_t pos;
  bool write, zero, rotate;
};

// All lanes of a wave call this together, their rows in ascending order.
template <typename T, bool APPEND, typename I>
__device__ __forceinline__ Target<T> target_of(const HeadArgs& a, const Row<T, I>& r, bool live) {
  Target<T> o;
  const int kind = r.kind;
  o.y = static_cast<T*>(AK_PICK(y)) + steps(r.h, AK_PICK(yh));
  o.rotate = kind < 2;
  o.zero = false;
  o.write = live;
  if constexpr (!APPEND) {
    o.pos = position_of(a, r.token);
    o.y += steps(r.token, AK_PICK(yt));
  } else {
    const int token = (int)r.token, b = sequence_of(a.seq, token);
    int pos = -1;
    if (b >= 0) {
      int first, count;
      sequence_tokens(a.seq, b, first, count);
      pos = max(a.seq.lengths[b], 0) - (count - (token - first));
    }
    o.pos = pos;
    if (kind == 0) {
      o.y += steps(r.token, a.r[0].yt);
      o.zero = b < 0;
      o.write = live && (b >= 0 || a.zero_tail);
    } else {
      int page = -1;
      uint32_t slot = 0;
      if (pos >= 0) {
        const uint32_t i = a.by_page(pos);
        slot = pos - i * (uint32_t)a.page_size;
        if (i < a.max_pages) page = a.pages[b * a.ld_pages + i];
      }
      o.write = live && page >= 0 && page < a.n_pages;
      if (o.write) o.y += steps((I)page, AK_PICK(yt)) + steps((I)slot, AK_PICK(ys));
    }
  }
  return o;
}
#undef AK_PICK

// Rows of whole vectors of VE elements: aligned to them, dim a multiple of one and the
// turned part of two. The widest that fits, 16, 8 or 4 bytes: of [8, 1024, 32 + 8, 128]
// bf16 with all or 64, 56 and 44 elements turned 28 (6.0 TB/s), 34 and 57 us, a wave a
// row 94; normed and back 88, 105 and 168 for 541. Prompts of 9730 tokens, 32 + 8 + 8
// heads of 128 fp16, normed into a cache 50 us (4.9 TB/s). A decode step is one launch
// of 4 us. Two or four rows a thread at a time, or fewer workgroups that read a row
// ahead: the same or slower.
template <typename T, int VE, bool NORM, bool APPEND>
__global__ void __launch_bounds__(kThreads) heads_kernel(HeadArgs a) {
  const int lpr = 1 << a.lpr_log2, per = kThreads >> a.lpr_log2;
  const int u = threadIdx.x & (lpr - 1);
  const Unit<VE> unit(u, a);
  const uint32_t total = (uint32_t)a.total;  // (and a walk's step more stays in 32 bits)
  for (uint32_t base = blockIdx.x * per; base < total; base += gridDim.x * per) {
    const uint32_t row = base + (threadIdx.x >> a.lpr_log2);
    const Row<T, uint32_t> from = row_of<T, APPEND>(a, min(row, total - 1));
    Vec<T, VE> v0, v1;
    v0.u = v1.u = typename Vec<T, VE>::W{};
    if (unit.has0) v0 = load_vec<VE>(from.x + unit.off0);
    if (unit.has1) v1 = load_vec<VE>(from.x + unit.off1);
    const Target<T> o = target_of<T, APPEND>(a, from, row < total);  // (its searches while the loads are on their way)
    if (!NORM && APPEND && !o.rotate) {  // values are copied
      if (o.write && unit.has0) store_vec(o.y + unit.off0, v0);
      if (o.write && unit.has1) store_vec(o.y + unit.off1, v1);
      continue;
    }
    float p[VE], q[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      p[e] = to_f32(v0.e[e]);
      q[e] = to_f32(v1.e[e]);
    }
    if constexpr (NORM) {
      float ss = 0.0f;
#pragma unroll
      for (int e = 0; e < VE; ++e) ss = fmaf(p[e], p[e], fmaf(q[e], q[e], ss));
      ss = lanes_sum(ss, a.lpr_log2);
      if (from.w != nullptr) {
        const float inv = 1.0f / sqrtf(ss * a.by_dim + a.eps);
        Vec<T, VE> w0, w1;
        w0.u = w1.u = typename Vec<T, VE>::W{};
        if (unit.has0) w0 = load_vec<VE>(from.w + unit.off0);
        if (unit.has1) w1 = load_vec<VE>(from.w + unit.off1);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          p[e] = p[e] * inv * to_f32(w0.e[e]);
          q[e] = q[e] * inv * to_f32(w1.e[e]);
        }
      }
    }
    if (unit.turned && o.rotate) {
      float c[VE], s[VE];
      load_angles<VE, !APPEND>(a, o.pos, u, c, s);
      turn<VE>(p, q, c, s, a.interleaved);
    }
    if (o.write) {
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        v0.e[e] = from_f32<T>(p[e]);
        v1.e[e] = from_f32<T>(q[e]);
      }
      if (APPEND && o.zero) v0.u = v1.u = typename Vec<T, VE>::W{};
      if (!APPEND && a.past) {
        if (unit.has0) store_past(o.y + unit.off0, v0);
        if (unit.has1) store_past(o.y + unit.off1, v1);
      } else {
        if (unit.has0) store_vec(o.y + unit.off0, v0);
        if (unit.has1) store_vec(o.y + unit.off1, v1);
      }
    }
  }
}

// Element i of a head's pair list: its two places.
__device__ __forceinline__ void pair_at(const HeadArgs& a, int i, int& e0, int& e1) {
  e0 = a.interleaved ? 2 * i : i;
  e1 = a.interleaved ? 2 * i + 1 : a.rotary / 2 + i;
}

__device__ __forceinline__ void angle_at(const HeadArgs& a, int64_t pos, int i, float& c, float& s) {
  c = s = __builtin_nanf("");
  if (pos >= 0 && pos < a.table_rows) {
    c = a.table[pos * a.rotary + i];
    s = a.table[pos * a.rotary + a.rotary / 2 + i];
    if (a.inverse) s = -s;
  }
}

// Every other row: a wave each, one element or pair a lane at a time. Bound by its narrow
// loads: [8, 1024, 32 + 8, 66] bf16 with 22 elements turned takes 89 us, forward and back with
// the norm 405.
template <typename T, bool NORM, bool APPEND, typename I>
__global__ void __launch_bounds__(kThreads) heads_any_kernel(HeadArgs a) {
  const int lane = threadIdx.x & 63;
  const I total = (I)a.total;
  for (I base = (I)blockIdx.x * 4; base < total; base += (I)gridDim.x * 4) {
    const I row = base + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // (places are the wave's: scalar work)
    const Row<T, I> from = row_of<T, APPEND>(a, min(row, total - 1));
    const Target<T> o = target_of<T, APPEND>(a, from, row < total);
    float inv = 1.0f;
    const bool norm = NORM && from.w != nullptr;
    if (norm) {
      float ss = 0.0f;
      for (int d = lane; d < a.dim; d += 64) {
        const float x = to_f32(from.x[d]);
        ss = fmaf(x, x, ss);
      }
      inv = 1.0f / sqrtf(wave_sum(ss) / (float)a.dim + a.eps);
    }
    if (!o.write) continue;
    auto value = [&](int d) {
      const float x = to_f32(from.x[d]);
      return norm ? x * inv * to_f32(from.w[d]) : x;
    };
    const int turned = o.rotate ? a.rotary : 0;
    for (int i = lane; i < turned / 2; i += 64) {
      int e0, e1;
      pair_at(a, i, e0, e1);
      float c, s;
      angle_at(a, o.pos, i, c, s);
      const float x0 = value(e0), x1 = value(e1);
      o.y[e0] = from_f32<T>(o.zero ? 0.0f : x0 * c - x1 * s);
      o.y[e1] = from_f32<T>(o.zero ? 0.0f : x1 * c + x0 * s);
    }
    for (int d = turned + lane; d < a.dim; d += 64) o.y[d] = from_f32<T>(o.zero ? 0.0f : value(d));
  }
}

// ---------------------------------------------------------------------------
// Backward of the norm with the rotation
// ---------------------------------------------------------------------------
struct GradRows {
  const void *x, *g, *w;
  void* dx;              // dense [tokens, heads, dim]
  void* dw;              // [dim] of the element type, or NULL
  int64_t so, si, sh;    // of x
  int64_t go, gi, gh;    // of g
  int64_t heads, rows;
  int first_block, blocks;
  Divisor by_heads;
};

struct GradArgs {
  GradRows r[2];
  HeadArgs h;            // the angles
  float* part;           // [blocks of both][dim]
};

template <typename T>
struct GradRow {
  const T *x, *g;
  int64_t pos;
};

template <typename T, typename I>
__device__ __forceinline__ GradRow<T> grad_row_of(const HeadArgs& a, const GradRows& r, I row) {
  const I token = quotient(row, r.heads, r.by_heads), h = row - token * (I)r.heads;
  I outer = 0, in = token;
  if (a.inner < a.tokens) {
    outer = quotient(token, a.inner, a.by_inner);
    in = token - outer * (I)a.inner;
  }
  return {static_cast<const T*>(r.x) + steps(outer, r.so) + steps(in, r.si) + steps(h, r.sh),
          static_cast<const T*>(r.g) + steps(outer, r.go) + steps(in, r.gi) + steps(h, r.gh), position_of(a, token)};
}

// A workgroup walks rows of one tensor; its lanes keep their unit, so the weight's
// gradient gathers in registers, then over the workgroup's rows in LDS, then over
// the workgroups in grad_weight_kernel: fixed orders throughout. [8, 1024, 32 + 8,
// 128] bf16 43 us (5.8 TB/s) and 4 for the weights, of 88 forward and back. The
// registers are held to 128 for four workgroups a CU: with three it was 117 for 97.
template <typename T, int VE>
__global__ void __launch_bounds__(kThreads, 4) heads_bwd_kernel(GradArgs ga) {
  __shared__ float gather[kThreads * 2 * VE];
  const HeadArgs& a = ga.h;
  const bool second = (int)blockIdx.x >= ga.r[1].first_block;
  const GradRows r = second ? ga.r[1] : ga.r[0];
  const int lpr = 1 << a.lpr_log2, per = kThreads >> a.lpr_log2;
  const int u = threadIdx.x & (lpr - 1), slot = threadIdx.x >> a.lpr_log2;
  const Unit<VE> unit(u, a);
  const T* w = static_cast<const T*>(r.w);
  float w0[VE], w1[VE], d0[VE], d1[VE];
  {
    Vec<T, VE> v0, v1;
    v0.u = v1.u = typename Vec<T, VE>::W{};
    if (unit.has0) v0 = load_vec<VE>(w + unit.off0);
    if (unit.has1) v1 = load_vec<VE>(w + unit.off1);
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      w0[e] = to_f32(v0.e[e]);
      w1[e] = to_f32(v1.e[e]);
      d0[e] = d1[e] = 0.0f;
    }
  }
  const uint32_t rows = (uint32_t)r.rows;
  for (uint32_t base = (blockIdx.x - r.first_block) * per; base < rows; base += r.blocks * per) {
    const uint32_t row = base + slot;
    const bool live = row < rows;
    const GradRow<T> o = grad_row_of<T>(a, r, min(row, rows - 1));
    Vec<T, VE> x0, x1, g0, g1;
    x0.u = x1.u = g0.u = g1.u = typename Vec<T, VE>::W{};
    if (live && unit.has0) {
      x0 = load_vec<VE>(o.x + unit.off0);
      g0 = load_vec<VE>(o.g + unit.off0);
    }
    if (live && unit.has1) {
      x1 = load_vec<VE>(o.x + unit.off1);
      g1 = load_vec<VE>(o.g + unit.off1);
    }
    float z0[VE], z1[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      z0[e] = to_f32(g0.e[e]);
      z1[e] = to_f32(g1.e[e]);
    }
    if (unit.turned) {
      float c[VE], s[VE];
      load_angles<VE, true>(a, o.pos, u, c, s);
      turn<VE>(z0, z1, c, s, a.interleaved);
    }
    float ss = 0.0f, gx = 0.0f;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const float a0 = to_f32(x0.e[e]), a1 = to_f32(x1.e[e]);
      ss = fmaf(a0, a0, fmaf(a1, a1, ss));
      gx = fmaf(z0[e] * w0[e], a0, fmaf(z1[e] * w1[e], a1, gx));
    }
    ss = lanes_sum(ss, a.lpr_log2);
    gx = lanes_sum(gx, a.lpr_log2);
    if (!live) continue;
    const float inv = 1.0f / sqrtf(ss * a.by_dim + a.eps);
    const float back = inv * (gx * a.by_dim);  // (of order one, as n is, whatever the size of x)
    Vec<T, VE> y0, y1;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const float n0 = to_f32(x0.e[e]) * inv, n1 = to_f32(x1.e[e]) * inv;
      y0.e[e] = from_f32<T>(inv * fmaf(z0[e], w0[e], -(n0 * back)));
      y1.e[e] = from_f32<T>(inv * fmaf(z1[e], w1[e], -(n1 * back)));
      d0[e] = fmaf(z0[e], n0, d0[e]);
      d1[e] = fmaf(z1[e], n1, d1[e]);
    }
    T* y = static_cast<T*>(r.dx) + steps(row, a.dim);
    if (a.past) {
      if (unit.has0) store_past(y + unit.off0, y0);
      if (unit.has1) store_past(y + unit.off1, y1);
    } else {
      if (unit.has0) store_vec(y + unit.off0, y0);
      if (unit.has1) store_vec(y + unit.off1, y1);
    }
  }
  if (r.dw == nullptr) return;
  // gather[element of the unit][thread]; then column by column over the row slots
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    gather[e * kThreads + threadIdx.x] = d0[e];
    gather[(VE + e) * kThreads + threadIdx.x] = d1[e];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < lpr * 2 * VE; i += kThreads) {
    const int lane_u = i & (lpr - 1), e = i >> a.lpr_log2;
    const Unit<VE> q(lane_u, a);
    const int col = e < VE ? q.off0 + e : q.off1 + e - VE;
    if (col >= a.dim) continue;
    float sum = 0.0f;
    for (int s = 0; s < per; ++s) sum += gather[e * kThreads + s * lpr + lane_u];
    ga.part[(int64_t)blockIdx.x * a.dim + col] = sum;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) heads_bwd_any_kernel(GradArgs ga) {
  __shared__ float gather[4][kMaxHeadDim];
  const HeadArgs& a = ga.h;
  const bool second = (int)blockIdx.x >= ga.r[1].first_block;
  const GradRows r = second ? ga.r[1] : ga.r[0];
  const T* w = static_cast<const T*>(r.w);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  float* mine = gather[wave];
  for (int d = lane; d < a.dim; d += 64) mine[d] = 0.0f;
  __syncthreads();
  for (int64_t row = (int64_t)((int)blockIdx.x - r.first_block) * 4 + wave; row < r.rows; row += (int64_t)r.blocks * 4) {
    const GradRow<T> o = grad_row_of<T>(a, r, row);
    // dz of pair i, or of the element rotary + (i - rotary / 2) past the pairs
    auto pair = [&](int i, int& e0, int& e1, float& z0, float& z1) {
      if (i < a.rotary / 2) {
        pair_at(a, i, e0, e1);
        float c, s;
        angle_at(a, o.pos, i, c, s);
        const float y0 = to_f32(o.g[e0]), y1 = to_f32(o.g[e1]);
        z0 = y0 * c - y1 * s;
        z1 = y1 * c + y0 * s;
      } else {
        e0 = a.rotary / 2 + i;
        e1 = -1;
        z0 = to_f32(o.g[e0]);
        z1 = 0.0f;
      }
    };
    const int n = a.dim - a.rotary / 2;
    float ss = 0.0f, gx = 0.0f;
    for (int i = lane; i < n; i += 64) {
      int e0, e1;
      float z0, z1;
      pair(i, e0, e1, z0, z1);
      const float x0 = to_f32(o.x[e0]), x1 = e1 >= 0 ? to_f32(o.x[e1]) : 0.0f, w1 = e1 >= 0 ? to_f32(w[e1]) : 0.0f;
      ss = fmaf(x0, x0, fmaf(x1, x1, ss));
      gx = fmaf(z0 * to_f32(w[e0]), x0, fmaf(z1 * w1, x1, gx));
    }
    ss = wave_sum(ss);
    gx = wave_sum(gx);
    const float inv = 1.0f / sqrtf(ss / (float)a.dim + a.eps);
    const float back = inv * (gx / (float)a.dim);  // (of order one, as n is, whatever the size of x)
    T* y = static_cast<T*>(r.dx) + row * a.dim;
    for (int i = lane; i < n; i += 64) {
      int e0, e1;
      float z0, z1;
      pair(i, e0, e1, z0, z1);
      const float n0 = to_f32(o.x[e0]) * inv;
      y[e0] = from_f32<T>(inv * fmaf(z0, to_f32(w[e0]), -(n0 * back)));
      mine[e0] = fmaf(z0, n0, mine[e0]);
      if (e1 >= 0) {
        const float n1 = to_f32(o.x[e1]) * inv;
        y[e1] = from_f32<T>(inv * fmaf(z1, to_f32(w[e1]), -(n1 * back)));
        mine[e1] = fmaf(z1, n1, mine[e1]);
      }
    }
  }
  __syncthreads();
  if (r.dw == nullptr) return;
  for (int d = threadIdx.x; d < a.dim; d += kThreads)
    ga.part[(int64_t)blockIdx.x * a.dim + d] = gather[0][d] + gather[1][d] + gather[2][d] + gather[3][d];
}

// The weights' gradients from the workgroups' parts: 16 columns a workgroup, 64
// threads each.
template <typename T>
__global__ void __launch_bounds__(1024) grad_weight_kernel(GradArgs ga) {
  __shared__ float sums[64][17];
  const int which = blockIdx.y;
  const int first = which ? ga.r[1].first_block : ga.r[0].first_block, n = which ? ga.r[1].blocks : ga.r[0].blocks;
  T* dw = static_cast<T*>(which ? ga.r[1].dw : ga.r[0].dw);
  if (dw == nullptr) return;
  const int c = threadIdx.x & 15, col = (int)blockIdx.x * 16 + c, group = threadIdx.x >> 4;
  const int dim = ga.h.dim;
  float sum = 0.0f;
  if (col < dim) {
#pragma unroll 4
    for (int i = group; i < n; i += 64) sum += ga.part[(int64_t)(first + i) * dim + col];
  }
  sums[group][c] = sum;
  __syncthreads();
  if (threadIdx.x < 256) {  // four groups each, then the 16 sums of a column, which a wave holds
    sum = 0.0f;
    for (int i = 0; i < 4; ++i) sum += sums[4 * (threadIdx.x & 15) + i][threadIdx.x >> 4];
    sum = row16_sum(sum);
    const int out = (int)blockIdx.x * 16 + (threadIdx.x >> 4);
    if ((threadIdx.x & 15) == 0 && out < dim) dw[out] = from_f32<T>(sum);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
bool on(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Fewest lanes (a power of two) that hold a head in units; past 64 the head
// takes the other kernels.
int lanes_log2(int64_t dim, int64_t rotary, int ve) {
  const int64_t units = rotary / (2 * ve) + (dim - rotary + 2 * ve - 1) / (2 * ve);
  int l = 0;
  while (((int64_t)1 << l) < units) ++l;
  return l;
}

// Leading dimensions that fold into one: a token's place then needs no division.
template <typename... Strides>
void fold_tokens(int64_t& outer, int64_t& inner, Strides... so_si) {
  const auto each = [&](auto fn) { (fn(*so_si.first, *so_si.second), ...); };
  if (inner == 1) {
    each([](int64_t& so, int64_t& si) { si = so; });
    inner = outer;
    outer = 1;
  }
  bool one = true;
  each([&](int64_t& so, int64_t& si) { one = one && so == inner * si; });
  if (one) {
    inner *= outer;
    outer = 1;
  }
}

int check_heads(const char* name, int64_t dim, int64_t rotary, int64_t table_rows, const float* table, float eps, int dtype) {
  if (ak_dtype_size(dtype) == 0) return ak_set_error(AK_ERR_UNSUPPORTED, "%s: unsupported dtype code %d", name, dtype);
  if (dim < 1 || dim > kMaxHeadDim)
    return ak_set_error(AK_ERR_UNSUPPORTED, "%s: head dim %lld is not 1 to %lld", name, (long long)dim, (long long)kMaxHeadDim);
  if (rotary < 0 || rotary > dim || rotary % 2)
    return ak_set_error(AK_ERR_INVALID_ARG, "%s: rotary %lld is not an even number up to dim", name, (long long)rotary);
  if (rotary > 0 && (!table || table_rows < 1 || table_rows > INT64_MAX / 4 / rotary))
    return ak_set_error(AK_ERR_INVALID_ARG, "%s: no table of angles", name);
  if (!(eps >= 0.0f) || eps > 3.0e38f) return ak_set_error(AK_ERR_INVALID_ARG, "%s: eps must be finite and not negative", name);
  return AK_OK;
}

template <typename T, bool NORM, bool APPEND>
void launch_heads(HeadArgs& a, hipStream_t s) {
  // (2^30 rows, and the last step of a walk)
  bool narrow = a.total <= 1 << 30 && a.table_rows <= INT32_MAX;
  for (const HeadRows& r : a.r)
    for (int64_t st : {r.heads > 1 ? r.sh : 0, r.heads > 1 ? r.yh : 0, r.si, r.so, r.yt, r.ys}) narrow = narrow && st <= (int64_t)UINT32_MAX;
  const auto fits = [&](int w) {
    bool ok = a.dim % w == 0 && a.rotary % (2 * w) == 0 && on(a.table, std::min(w, 4) * 4) && lanes_log2(a.dim, a.rotary, w) <= 6;
    for (const HeadRows& r : a.r) {
      if (r.heads == 0) continue;
      for (const void* p : {r.x, (const void*)r.y, r.w}) ok = ok && on(p, w * (int)sizeof(T));
      for (int64_t st : {r.so, r.si, r.sh, r.yt, r.ys, r.yh}) ok = ok && st % w == 0;
    }
    return ok;
  };
  constexpr int VE = Vec16<T>::VE;
  const int w = !narrow ? 0 : fits(VE) ? VE : fits(VE / 2) ? VE / 2 : VE > 4 && fits(VE / 4) ? VE / 4 : 0;
  a.lpr_log2 = w ? lanes_log2(a.dim, a.rotary, w) : 6;
  a.by_heads = Divisor(a.all_heads);
  a.by_inner = Divisor(a.inner);
  a.by_positions = Divisor(a.n_positions);
  a.by_page = Divisor(a.page_size);
  a.by_dim = 1.0f / (float)a.dim;
  a.past = a.total > kL2Bytes / (a.dim * (int64_t)sizeof(T));
  const int64_t per = kThreads >> a.lpr_log2;
  const dim3 grid(row_grid((a.total + per - 1) / per)), block(kThreads);
  if (w == VE) heads_kernel<T, VE, NORM, APPEND><<<grid, block, 0, s>>>(a);
  else if (w == VE / 2) heads_kernel<T, VE / 2, NORM, APPEND><<<grid, block, 0, s>>>(a);
  else if (VE > 4 && w == VE / 4) heads_kernel<T, (VE > 4 ? VE / 4 : 2), NORM, APPEND><<<grid, block, 0, s>>>(a);
  else if (narrow) heads_any_kernel<T, NORM, APPEND, uint32_t><<<grid, block, 0, s>>>(a);
  else heads_any_kernel<T, NORM, APPEND, int64_t><<<grid, block, 0, s>>>(a);
}

template <bool APPEND>
void dispatch_heads(HeadArgs& a, bool norm, int dtype, hipStream_t s) {
  auto go = [&](auto t) {
    using T = decltype(t);
    if (norm) launch_heads<T, true, APPEND>(a, s);
    else launch_heads<T, false, APPEND>(a, s);
  };
  if (dtype == AK_DTYPE_F32) go(float());
  else if (dtype == AK_DTYPE_F16) go(f16());
  else go(bf16());
}

constexpr int64_t kGradBlocks = 1024;

// Workgroups of the backward for queries and keys: by their heads, at least one
// where there are any, at most one for each group of rows.
void grad_blocks(int64_t tokens, int64_t q_heads, int64_t k_heads, int64_t* bq, int64_t* bk) {
  const int64_t all = q_heads + k_heads;
  auto share = [&](int64_t heads) {
    if (heads == 0 || tokens == 0) return (int64_t)0;
    const int64_t want = (int64_t)((double)kGradBlocks * (double)heads / (double)all + 0.5);
    // (a workgroup of the vector form takes 4 rows at least)
    const int64_t rows = tokens > (kGradBlocks * 4) / heads ? kGradBlocks * 4 : tokens * heads;
    return std::max((int64_t)1, std::min(want, (rows + 3) / 4));
  };
  *bq = share(q_heads);
  *bk = share(k_heads);
}

}  // namespace
}  // namespace ak

extern "C" int ak_qk_norm_rotary_fwd(const void* q, const void* k, const void* q_weight, const void* k_weight,
                                     const float* table, const void* positions, void* q_out, void* k_out, int64_t outer,
                                     int64_t inner, int64_t q_heads, int64_t k_heads, int64_t dim, int64_t rotary,
                                     int64_t table_rows, int64_t n_positions, int64_t q_so, int64_t q_si, int64_t q_sh,
                                     int64_t k_so, int64_t k_si, int64_t k_sh, float eps, int flags, int dtype, void* stream) {
  const char* name = "ak_qk_norm_rotary_fwd";
  int rc = ak::check_heads(name, dim, rotary, table_rows, table, eps, dtype);
  if (rc) return rc;
  const int esz = ak_dtype_size(dtype);
  if (outer < 0 || inner < 0 || q_heads < 0 || k_heads < 0 || q_heads > INT32_MAX || k_heads > INT32_MAX ||
      !ak::extent_ok(outer, q_so, inner, q_si, q_heads, q_sh, dim, esz) ||
      !ak::extent_ok(outer, k_so, inner, k_si, k_heads, k_sh, dim, esz) ||
      (__int128)outer * inner * (q_heads + k_heads) * dim > INT64_MAX / esz)
    return ak_set_error(AK_ERR_INVALID_ARG, "%s: bad shape or strides", name);
  const int64_t tokens = outer * inner;
  if (tokens == 0 || q_heads + k_heads == 0) return AK_OK;
  if (n_positions < 1) return ak_set_error(AK_ERR_INVALID_ARG, "%s: no positions", name);
  if ((q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out)) || (q_heads && k_heads && !q_weight != !k_weight))
    return ak_set_error(AK_ERR_INVALID_ARG, "%s: null pointer", name);
  ak::fold_tokens(outer, inner, std::make_pair(&q_so, &q_si), std::make_pair(&k_so, &k_si));
  ak::HeadArgs a{};
  a.r[0] = {q, q_out, q_weight, q_so, q_si, q_sh, q_heads * dim, 0, dim, q_heads};
  a.r[1] = {k, k_out, k_weight, k_so, k_si, k_sh, k_heads * dim, 0, dim, k_heads};
  a.table = table;
  a.positions = positions;
  a.tokens = tokens;
  a.inner = inner;
  a.n_positions = std::min(n_positions, tokens);
  a.table_rows = table_rows;
  a.all_heads = q_heads + k_heads;
  a.total = tokens * a.all_heads;
  a.dim = (int)dim;
  a.rotary = (int)rotary;
  a.interleaved = (flags & AK_ROTARY_INTERLEAVED) != 0;
  a.inverse = (flags & AK_ROTARY_INVERSE) != 0;
  a.pos64 = (flags & AK_POSITIONS_I64) != 0;
  a.eps = eps;
  ak::dispatch_heads<false>(a, (q_heads && q_weight) || (k_heads && k_weight), dtype, ak_stream(stream));
  return ak_check_launch(name);
}

extern "C" size_t ak_qk_norm_rotary_bwd_workspace_bytes(int64_t tokens, int64_t q_heads, int64_t k_heads, int64_t dim) {
  if (tokens <= 0 || q_heads < 0 || k_heads < 0 || dim <= 0) return 0;
  int64_t bq, bk;
  ak::grad_blocks(tokens, q_heads, k_heads, &bq, &bk);
  return (size_t)(bq + bk) * (size_t)dim * sizeof(float);
}

extern "C" int ak_qk_norm_rotary_bwd(const void* q, const void* k, const void* q_weight, const void* k_weight,
                                     const float* table, const void* positions, const void* grad_q_out,
                                     const void* grad_k_out, void* grad_q, void* grad_k, void* grad_q_weight,
                                     void* grad_k_weight, void* workspace, size_t workspace_bytes, int64_t outer,
                                     int64_t inner, int64_t q_heads, int64_t k_heads, int64_t dim, int64_t rotary,
                                     int64_t table_rows, int64_t n_positions, int64_t q_so, int64_t q_si, int64_t q_sh,
                                     int64_t k_so, int64_t k_si, int64_t k_sh, int64_t gq_so, int64_t gq_si, int64_t gq_sh,
                                     int64_t gk_so, int64_t gk_si, int64_t gk_sh, float eps, int flags, int dtype,
                                     void* stream) {
  const char* name = "ak_qk_norm_rotary_bwd";
  int rc = ak::check_heads(name, dim, rotary, table_rows, table, eps, dtype);
  if (rc) return rc;
  const int esz = ak_dtype_size(dtype);
  if (outer < 0 || inner < 0 || q_heads < 0 || k_heads < 0 || q_heads > INT32_MAX || k_heads > INT32_MAX ||
      !ak::extent_ok(outer, q_so, inner, q_si, q_heads, q_sh, dim, esz) ||
      !ak::extent_ok(outer, k_so, inner, k_si, k_heads, k_sh, dim, esz) ||
      !ak::extent_ok(outer, gq_so, inner, gq_si, q_heads, gq_sh, dim, esz) ||
      !ak::extent_ok(outer, gk_so, inner, gk_si, k_heads, gk_sh, dim, esz) ||
      (__int128)outer * inner * (q_heads + k_heads) * dim > INT64_MAX / esz)
    return ak_set_error(AK_ERR_INVALID_ARG, "%s: bad shape or strides", name);
  const int64_t tokens = outer * inner;
  if (tokens > 0 && n_positions < 1) return ak_set_error(AK_ERR_INVALID_ARG, "%s: no positions", name);
  const bool some = tokens > 0;
  if ((some && q_heads && (!q || !q_weight || !grad_q_out || !grad_q)) || (some && k_heads && (!k || !k_weight || !grad_k_out || !grad_k)))
    return ak_set_error(AK_ERR_INVALID_ARG, "%s: null pointer", name);
  const size_t need = ak_qk_norm_rotary_bwd_workspace_bytes(tokens, q_heads, k_heads, dim);
  if (workspace_bytes < need || (need && (!workspace || !ak::aligned16(workspace))))
    return ak_set_error(AK_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed (16-byte aligned)", name, workspace_bytes, need);
  ak::fold_tokens(outer, inner, std::make_pair(&q_so, &q_si), std::make_pair(&k_so, &k_si),
                  std::make_pair(&gq_so, &gq_si), std::make_pair(&gk_so, &gk_si));
  ak::GradArgs g{};
  int64_t bq, bk;
  ak::grad_blocks(tokens, q_heads, k_heads, &bq, &bk);
  g.r[0] = {q, grad_q_out, q_weight, grad_q, grad_q_weight, q_so, q_si, q_sh, gq_so, gq_si, gq_sh, q_heads,
            tokens * q_heads, 0, (int)bq};
  g.r[1] = {k, grad_k_out, k_weight, grad_k, grad_k_weight, k_so, k_si, k_sh, gk_so, gk_si, gk_sh, k_heads,
            tokens * k_heads, (int)bq, (int)bk};
  g.part = static_cast<float*>(workspace);
  ak::HeadArgs& a = g.h;
  a.table = table;
  a.positions = positions;
  a.tokens = tokens;
  a.inner = inner;
  a.n_positions = std::min(n_positions, tokens);
  a.table_rows = table_rows;
  a.dim = (int)dim;
  a.rotary = (int)rotary;
  a.interleaved = (flags & AK_ROTARY_INTERLEAVED) != 0;
  a.inverse = 1;
  a.pos64 = (flags & AK_POSITIONS_I64) != 0;
  a.eps = eps;
  hipStream_t s = ak_stream(stream);
  auto go = [&](auto t) {
    using T = decltype(t);
    bool narrow = table_rows <= INT32_MAX;
    for (ak::GradRows& r : g.r) {
      r.by_heads = ak::Divisor(r.heads);
      narrow = narrow && r.rows <= 1 << 30;
      for (int64_t st : {r.so, r.si, r.sh, r.go, r.gi, r.gh}) narrow = narrow && (r.heads == 0 || st <= (int64_t)UINT32_MAX);
    }
    const auto fits = [&](int w) {
      bool ok = dim % w == 0 && rotary % (2 * w) == 0 && ak::on(table, std::min(w, 4) * 4) && ak::lanes_log2(dim, rotary, w) <= 6;
      for (const ak::GradRows& r : g.r) {
        if (r.heads == 0) continue;
        for (const void* p : {r.x, r.g, r.w, (const void*)r.dx}) ok = ok && ak::on(p, w * (int)sizeof(T));
        for (int64_t st : {r.so, r.si, r.sh, r.go, r.gi, r.gh}) ok = ok && st % w == 0;
      }
      return ok;
    };
    constexpr int VE = ak::Vec16<T>::VE;
    const int w = !narrow ? 0 : fits(VE) ? VE : fits(VE / 2) ? VE / 2 : VE > 4 && fits(VE / 4) ? VE / 4 : 0;
    if (w) a.lpr_log2 = ak::lanes_log2(dim, rotary, w);
    a.by_inner = ak::Divisor(a.inner);
    a.by_positions = ak::Divisor(a.n_positions);
    a.by_dim = 1.0f / (float)dim;
    a.past = tokens * (q_heads + k_heads) > ak::kL2Bytes / (dim * (int64_t)sizeof(T));
    if (bq + bk > 0) {
      const dim3 grid((unsigned)(bq + bk)), block(ak::kThreads);
      if (w == VE) ak::heads_bwd_kernel<T, VE><<<grid, block, 0, s>>>(g);
      else if (w == VE / 2) ak::heads_bwd_kernel<T, VE / 2><<<grid, block, 0, s>>>(g);
      else if (VE > 4 && w == VE / 4) ak::heads_bwd_kernel<T, (VE > 4 ? VE / 4 : 2)><<<grid, block, 0, s>>>(g);
      else ak::heads_bwd_any_kernel<T><<<grid, block, 0, s>>>(g);
    }
    if (grad_q_weight || grad_k_weight)
      ak::grad_weight_kernel<T><<<dim3((unsigned)((dim + 15) / 16), 2), dim3(1024), 0, s>>>(g);
  };
  if (dtype == AK_DTYPE_F32) go(float());
  else if (dtype == AK_DTYPE_F16) go(ak::f16());
  else go(ak::bf16());
  return ak_check_launch(name);
}

extern "C" int ak_paged_append(const void* q, const void* k, const void* v, const void* q_weight, const void* k_weight,
                               const float* table, void* q_out, void* k_cache, void* v_cache, const int32_t* page_table,
                               const int32_t* lengths, const int32_t* starts, int64_t tokens, int64_t batch, int64_t q_heads,
                               int64_t kv_heads, int64_t dim, int64_t rotary, int64_t table_rows, int64_t n_pages,
                               int64_t page_size, int64_t max_pages, int64_t ld_pages, int64_t q_st, int64_t q_sh,
                               int64_t k_st, int64_t k_sh, int64_t v_st, int64_t v_sh, int64_t qo_st, int64_t qo_sh,
                               int64_t kc_sp, int64_t kc_ss, int64_t kc_sh, int64_t vc_sp, int64_t vc_ss, int64_t vc_sh,
                               float eps, int flags, int dtype, void* stream) {
  const char* name = "ak_paged_append";
  int rc = ak::check_heads(name, dim, rotary, table_rows, table, eps, dtype);
  if (rc) return rc;
  const int esz = ak_dtype_size(dtype);
  rc = ak::check_paged(name, tokens, batch, n_pages, page_size, max_pages, ld_pages, starts, lengths, page_table);
  if (rc) return rc;
  if (q_heads < 0 || kv_heads < 1 || q_heads > INT32_MAX / 4 || kv_heads > INT32_MAX / 4 ||
      !ak::extent_ok(1, 0, tokens, q_st, q_heads, q_sh, dim, esz) || !ak::extent_ok(1, 0, tokens, qo_st, q_heads, qo_sh, dim, esz) ||
      !ak::extent_ok(1, 0, tokens, k_st, kv_heads, k_sh, dim, esz) || !ak::extent_ok(1, 0, tokens, v_st, kv_heads, v_sh, dim, esz) ||
      !ak::extent_ok(n_pages, kc_sp, page_size, kc_ss, kv_heads, kc_sh, dim, esz) ||
      !ak::extent_ok(n_pages, vc_sp, page_size, vc_ss, kv_heads, vc_sh, dim, esz) ||
      (__int128)tokens * (q_heads + 2 * kv_heads) > INT64_MAX / 4096)
    return ak_set_error(AK_ERR_INVALID_ARG, "%s: bad shape or strides", name);
  if (tokens == 0) return AK_OK;
  if ((q_heads && (!q || !q_out)) || !k || !v || (n_pages && (!k_cache || !v_cache)))
    return ak_set_error(AK_ERR_INVALID_ARG, "%s: null pointer", name);
  ak::HeadArgs a{};
  a.r[0] = {q, q_out, q_weight, 0, q_st, q_sh, qo_st, 0, qo_sh, q_heads};
  a.r[1] = {k, k_cache, k_weight, 0, k_st, k_sh, kc_sp, kc_ss, kc_sh, kv_heads};
  a.r[2] = {v, v_cache, nullptr, 0, v_st, v_sh, vc_sp, vc_ss, vc_sh, kv_heads};
  a.table = table;
  a.tokens = a.inner = a.n_positions = tokens;
  a.table_rows = table_rows;
  a.all_heads = q_heads + 2 * kv_heads;
  a.total = tokens * a.all_heads;
  a.dim = (int)dim;
  a.rotary = (int)rotary;
  a.interleaved = (flags & AK_ROTARY_INTERLEAVED) != 0;
  a.zero_tail = (flags & AK_ZERO_OTHER_ROWS) != 0;
  a.eps = eps;
  a.seq = {starts, lengths, batch, tokens, starts ? 0 : tokens / batch};
  a.pages = page_table;
  a.n_pages = n_pages;
  a.page_size = page_size;
  a.max_pages = max_pages;
  a.ld_pages = ld_pages;
  ak::dispatch_heads<true>(a, (q_heads && q_weight) || k_weight, dtype, ak_stream(stream));
  return ak_check_launch(name);
}
