// Rows of logits read once for their softmax statistics: shared by the token
// log probabilities (token_logprobs.hip) and the distillation loss
// (topk_distill.hip).
//
// With the score y = softcap tanh(x / softcap) (or x) and c2 = log2(e) /
// temperature, a row's statistics are its maximum m of y and
//   t = (y - m) c2,   s = sum 2^t,   u = sum 2^t t,
// so that ln p = ln2 (t - log2 s) and the entropy is ln2 (log2 s - u / s).
// y - m is formed before the product: it is exact at the maximum whatever the
// logits' size, where fma(y, c2, -m c2) would leave m c2's rounding in every
// exponent. All statistics are fp32.
//
// A row is cut into `segs` segments of `span` 16-byte vectors. One workgroup
// holds a segment in registers, packed, so that it crosses HBM once, 16 vectors
// a thread where it is that wide: with 8 in twice the threads, the same bytes in
// flight and twice the waves at each barrier, [8192, 50304] bf16 takes 233 us
// for 152 to 160, [4096, 50257] bf16 and fp16 123 for 84, the distillation step
// of [1999, 50257] fp32 262 for 216, [4096, 32768] bf16 with 64 alternatives 80
// for 76. One segment a row where rows fill the GPU and a row fits a workgroup;
// otherwise each segment leaves its (m, s, u) in a workspace and a second kernel
// joins them, as a decode step's few rows need every CU (plan below).
#pragma once

#include <algorithm>

#include "ak_common.h"

namespace ak {

typedef float f32x4_t __attribute__((ext_vector_type(4)));

// What the statistics mean: the capped, tempered logits.
struct ScoreParams {
  float cap, inv_cap;  // softcap (with CAP)
  float k2;            // 2 log2(e) / softcap
  float c2;            // log2(e) / temperature
  float inv_t;         // 1 / temperature
  int64_t ignore_index;
};

inline ScoreParams score_params(float temperature, float softcap, int64_t ignore_index) {
  ScoreParams p;
  p.cap = softcap;
  p.inv_cap = softcap > 0.0f ? 1.0f / softcap : 0.0f;
  p.k2 = softcap > 0.0f ? (float)(2.8853900817779268 / (double)softcap) : 0.0f;
  p.c2 = (float)(1.4426950408889634 / (double)temperature);
  p.inv_t = 1.0f / temperature;
  p.ignore_index = ignore_index;
  return p;
}

template <bool CAP>
__device__ __forceinline__ float score(const ScoreParams& p, float x) {
  return CAP ? p.cap * tanh_f32(x * p.inv_cap) : x;
}

// The score of one of a row's many logits of type T. Half-precision logits are
// rounded to 2^-9 or 2^-12 of themselves already, so their cap takes the short
// form cap - 2 cap r, r = 1 / (1 + exp(2 x / cap)), within 2^-22 cap of the exact
// one (5 instructions for tanh_f32's 14: the forward of [4096, 50257] bf16 with a
// softcap 129 -> 106 us).
template <typename T, bool CAP>
__device__ __forceinline__ float many_score(const ScoreParams& p, float x) {
  if constexpr (CAP && !std::is_same<T, float>::value)
    return fmaf(-2.0f * p.cap, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * p.k2)), p.cap);
  return score<CAP>(p, x);
}

// (m, s, u) of a row or a segment of one.
struct RowStats {
  float m, s, u;
};

// A row of -inf alone has no distribution: m = -inf, s = 0. (A row that holds
// a NaN or +inf has s = NaN.)
__device__ __forceinline__ bool empty_row(float m, float s) { return m == -INFINITY && s == 0.0f; }

// log2 s as the log probabilities take it (0 for an empty row, whose scores are -inf already).
__device__ __forceinline__ float log2_sum(const RowStats& r) {
  return empty_row(r.m, r.s) ? 0.0f : __builtin_amdgcn_logf(r.s);
}

// ln p of a score; l2: log2_sum. (In natural units: a mask of the type's
// lowest value stays in fp32's range, which its product with c2 would leave.) At
// most 0: under a softcap y and the row's sum come from two forms of the tanh.
__device__ __forceinline__ float log_prob(const ScoreParams& p, float y, float m, float l2) {
  const float lp = m == -INFINITY && y == -INFINITY ? y - l2 : (y - m) * p.inv_t - kLn2 * l2;
  return lp > 0.0f ? 0.0f : lp;  // (NaN stays)
}

__device__ __forceinline__ float row_entropy(const RowStats& r) {
  if (empty_row(r.m, r.s)) return 0.0f;
  const float h = kLn2 * (__builtin_amdgcn_logf(r.s) - r.u / r.s);
  return h < 0.0f ? 0.0f : h;  // one rounding below zero where one entry holds all
}

// Statistics of two parts of one row.
__device__ __forceinline__ RowStats join_stats(const ScoreParams& p, RowStats a, RowStats b) {
  const float m = fmaxf(a.m, b.m);
  RowStats r{m, 0.0f, 0.0f};
  auto add = [&](const RowStats& q) {
    if (q.s == 0.0f) return;
    const float d = (q.m - m) * p.c2;  // NaN for +inf maxima: the row's sum becomes NaN
    const float f = __builtin_amdgcn_exp2f(d);
    r.s += f * q.s;
    // f = 0 where a part vanishes beside the other: its d may be -inf
    r.u += f * (q.u + fmaxf(d, -1000.0f) * q.s);
  };
  add(a);
  add(b);
  return r;
}

__device__ __forceinline__ RowStats wave_join(const ScoreParams& p, RowStats st) {
  for (int off = 1; off < 64; off <<= 1) {
    const RowStats o{__shfl_xor(st.m, off, 64), __shfl_xor(st.s, off, 64), __shfl_xor(st.u, off, 64)};
    // the lower lane's part first, so that every lane ends with the same bits
    st = (threadIdx.x & off) ? join_stats(p, o, st) : join_stats(p, st, o);
  }
  return st;
}

// The largest element of a vector. In assembly, since fmaxf first quiets each
// operand that it does not know to be quiet (an instruction an element). A
// signalling NaN makes the result NaN, a quiet one is passed over; a row that
// holds either has a NaN sum. (The caller's next use is no lane permutation,
// which would need wait states that the compiler does not see here.)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float m;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(a), "v"(b), "v"(c));
  return m;
}
__device__ __forceinline__ float vec_max(const Vec16<float>& v) { return max3(max3(v.e[0], v.e[1], v.e[2]), v.e[3], v.e[3]); }
__device__ __forceinline__ float vec_max(const Vec16<bf16>& v) {
  auto lo = [&](int i) { return __builtin_bit_cast(float, v.u[i] << 16); };
  auto hi = [&](int i) { return __builtin_bit_cast(float, v.u[i] & 0xFFFF0000u); };
  return max3(max3(max3(max3(lo(0), hi(0), lo(1)), hi(1), lo(2)), hi(2), lo(3)), hi(3), hi(3));
}
__device__ __forceinline__ float vec_max(const Vec16<f16>& v) {
  uint32_t a, b;
  asm("v_pk_max_f16 %0, %1, %2" : "=v"(a) : "v"(v.u[0]), "v"(v.u[1]));
  asm("v_pk_max_f16 %0, %1, %2" : "=v"(b) : "v"(v.u[2]), "v"(v.u[3]));
  asm("v_pk_max_f16 %0, %1, %2" : "=v"(a) : "v"(a), "v"(b));
  const f16x2_t m = __builtin_bit_cast(f16x2_t, a);
  return max3((float)m[0], (float)m[1], (float)m[1]);
}

// A segment of a row in registers: TPR threads, VPT vectors each, and the
// elements around the row's vectors (at most 14, with the first segment) one
// to a thread.
template <typename T, int VPT, int TPR>
struct Segment {
  static constexpr int VE = Vec16<T>::VE;
  Vec16<T> raw[VPT];
  T xe;
  int nv, nx;  // vectors of the segment, single elements
  int col0;    // column of its first vector
  RowSplit<T> sp;

  // The thread's index, opaque to the compiler in each pass: the VPT offsets
  // and bounds derived from it would otherwise be held from pass to pass
  // beside the segment, and spill.
  static __device__ __forceinline__ int thread() {
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
  }

  __device__ __forceinline__ Segment(const T* __restrict__ row, int vocab, int seg, int span) : sp(row, vocab) {
    const int v0 = seg * span;
    nv = min(span, sp.nvec - v0);
    nx = seg == 0 ? sp.nx : 0;
    col0 = sp.head + v0 * VE;
    const int t = thread();
    xe = T(0.0f);
    if (t < nx) xe = row[sp.extra(t)];
    const T* rv = row + col0;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      raw[k].u = u32x4{0, 0, 0, 0};
      if (t + k * TPR < nv) raw[k] = load16_any_nt(rv + k * TPR * VE + (unsigned)(t * VE));
    }
  }

  // f(logit, column) of each element that this thread holds.
  template <typename F>
  __device__ __forceinline__ void each(F f) {
    const int t = thread();
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      if (t + k * TPR < nv) {
#pragma unroll
        for (int e = 0; e < VE; ++e) f(to_f32(raw[k].e[e]), col0 + (t + k * TPR) * VE + e);
      }
      keep_packed(raw[k]);
    }
    if (t < nx) f(to_f32(xe), sp.extra(t));
  }

  // This thread's largest logit (NaN ignored).
  __device__ __forceinline__ float largest() {
    const int t = thread();
    float m = t < nx ? to_f32(xe) : -INFINITY;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const float vm = vec_max(raw[k]);
      m = fmaxf(m, t + k * TPR < nv ? vm : -INFINITY);
      keep_packed(raw[k]);
    }
    return m;
  }

  // The same, and the maxima of the segment's groups of 2^SHIFT vectors, joined
  // over as many lanes. maxima: the segment's first group's place; group: what
  // this thread stores of them (store_groups): lane l of a group's lanes those
  // of the vectors l, l + 2^SHIFT, ...
  template <int SHIFT>
  static constexpr int kStored = SHIFT > 0 ? (VPT + (1 << SHIFT) - 1) >> SHIFT : 1;

  template <int SHIFT>
  __device__ __forceinline__ float largest_of_groups(float* __restrict__ maxima, float (&group)[kStored<SHIFT>]) {
    const int t = thread();
    float m = t < nx ? to_f32(xe) : -INFINITY;
    const int l = t & ((1 << SHIFT) - 1);
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const bool in = t + k * TPR < nv;
      float vm = vec_max(raw[k]);
      vm = in ? vm : -INFINITY;
      m = fmaxf(m, vm);
      if constexpr (SHIFT >= 3) {
        vm = fmaxf(vm, dpp<kDppXor1>(vm));
        vm = fmaxf(vm, dpp<kDppXor2>(vm));
        vm = fmaxf(vm, dpp<kDppHalfMirror>(vm));
      }
      if constexpr (SHIFT == 6) {
        vm = fmaxf(vm, dpp<kDppMirror>(vm));
        vm = fmaxf(vm, __shfl_xor(vm, 16, 64));
        vm = fmaxf(vm, __shfl_xor(vm, 32, 64));
      }
      if constexpr (SHIFT == 0) {
        if (in) maxima[t + k * TPR] = vm;
      } else {
        group[k >> SHIFT] = (k & ((1 << SHIFT) - 1)) == l ? vm : group[k >> SHIFT];
      }
      keep_packed(raw[k]);
    }
    return m;
  }

  template <int SHIFT>
  __device__ __forceinline__ void store_groups(float* __restrict__ maxima, const float (&group)[kStored<SHIFT>]) const {
    const int t = thread(), l = t & ((1 << SHIFT) - 1);
#pragma unroll
    for (int i = 0; i < kStored<SHIFT>; ++i) {
      const int k = (i << SHIFT) + l, v = (t & ~((1 << SHIFT) - 1)) + k * TPR;  // the group's first vector
      if (k < VPT && v < nv) maxima[v >> SHIFT] = group[i];
    }
  }

  // This thread's part of s and, with ENT, of u.
  template <bool CAP, bool ENT>
  __device__ __forceinline__ void sums(const ScoreParams& p, float m, float& s, float& u) {
    const float off = m == -INFINITY ? 0.0f : m;
    s = u = 0.0f;
    each([&](float x, int) {
      const float t = (many_score<T, CAP>(p, x) - off) * p.c2;
      const float e = __builtin_amdgcn_exp2f(t);
      s += e;
      // 2^t is 0 from -150 on, and t may be -inf there
      if constexpr (ENT) u = fmaf(e, fmaxf(t, -1000.0f), u);
    });
  }
};

// How rows are cut and held (host).
struct ScorePlan {
  int segs, span;  // segments a row, vectors a segment
};

constexpr int kSegVectors = 8192;            // most vectors of a segment: 512 threads x 16
constexpr int64_t kScoreVocab = 1 << 20;     // widest row
constexpr int kMaxTop = 256;                 // most alternatives

// One segment a row where there are rows for every CU. Fewer rows are cut so
// that about two workgroups a CU share the work, in segments of at least 256
// vectors (one a thread), whole multiples of 64.
inline ScorePlan score_plan(int64_t rows, int64_t vocab, int ve) {
  const int64_t nvec = std::max<int64_t>(1, vocab / ve);
  const int64_t least = (nvec + kSegVectors - 1) / kSegVectors;
  int64_t segs = least;
  if (rows < 256) segs = std::max(segs, std::min((512 + rows - 1) / rows, nvec / 256));
  const int64_t span = ((nvec + segs - 1) / segs + 63) / 64 * 64;
  return {(int)((nvec + span - 1) / span), (int)span};
}

// kernel<VPT, TPR> for a segment of `span` vectors.
#define AK_SEGMENT_DISPATCH(span, GO)    \
  do {                                   \
    if ((span) <= 256) GO(1, 256);       \
    else if ((span) <= 512) GO(2, 256);  \
    else if ((span) <= 1024) GO(4, 256); \
    else if ((span) <= 2048) GO(8, 256); \
    else if ((span) <= 4096) GO(16, 256);\
    else GO(16, 512);                    \
  } while (0)
// (waves a SIMD that the register budget is set for)
#define AK_SEGMENT_WAVES(VPT) ((VPT) == 16 ? 4 : (VPT) == 8 ? 6 : 1)

// ---------------------------------------------------------------------------
// Gradients: rows written whole from their statistics
// ---------------------------------------------------------------------------
constexpr int kGradThreads = 256;

// d(score / temperature) / d(logit), and the score (as many_score). The slope 1 -
// tanh^2 as 4 q / (1 + q)^2 with q = exp(2 x / cap): a difference from 1 would
// have nothing left where the cap is near. (q may be inf, r 0 then: q is held at
// 2^125, up to which r q is 1 and the slope keeps its digits.)
template <typename T, bool CAP>
__device__ __forceinline__ float score_and_slope(const ScoreParams& p, float x, float& slope) {
  if constexpr (CAP && !std::is_same<T, float>::value) {
    const float q = __builtin_amdgcn_exp2f(x * p.k2), r = __builtin_amdgcn_rcpf(1.0f + q);
    slope = 4.0f * p.inv_t * r * (r * fminf(q, 0x1p125f));
    return fmaf(-2.0f * p.cap, r, p.cap);
  }
  if constexpr (CAP) {
    const float a = x * p.inv_cap, q = fast_exp(-2.0f * fabsf(a)), r = __builtin_amdgcn_rcpf(1.0f + q);
    slope = 4.0f * p.inv_t * r * (r * q);
    return p.cap * tanh_f32(a);  // (the same exponential and reciprocal)
  }
  slope = p.inv_t;
  return x;
}

// The gradient of the row's vectors [v0, v1) and, with `ends`, of the elements
// around the vectors: g.many(x) of each logit, and g.patch(col, v - v0, o) may
// change a vector of results; g.one(x, col, i) of single element i. U vectors of
// a thread are loaded before the first is used.
template <typename T, bool NT, int U, typename G>
__device__ __forceinline__ void map_row(const T* __restrict__ row, T* __restrict__ out, int vocab, int v0, int v1,
                                        bool ends, const G& g) {
  constexpr int VE = Vec16<T>::VE;
  const RowSplit<T> sp(row, vocab);
  const int t = threadIdx.x;
  const T* rv = row + sp.head;
  T* ov = out + sp.head;
  if (v1 > sp.nvec) v1 = sp.nvec;
  auto ld = [](const T* q) { return NT ? load16_any_nt(q) : load16_any(q); };
  auto one = [&](const Vec16<T>& x, int v) {
    Vec16<T> o;
#pragma unroll
    for (int e = 0; e < VE; ++e) o.e[e] = from_f32<T>(g.many(to_f32(x.e[e])));
    g.patch(x, sp.head + v * VE, v - v0, o);
    if (NT) store16_any_nt(ov + (int64_t)v * VE, o);
    else store16_any(ov + (int64_t)v * VE, o);
  };
  int v = v0 + t;
  for (; U > 1 && v + (U - 1) * kGradThreads < v1; v += U * kGradThreads) {
    Vec16<T> x[U];
#pragma unroll
    for (int i = 0; i < U; ++i) x[i] = ld(rv + (int64_t)(v + i * kGradThreads) * VE);
#pragma unroll
    for (int i = 0; i < U; ++i) one(x[i], v + i * kGradThreads);
  }
  for (; v < v1; v += kGradThreads) one(ld(rv + (int64_t)v * VE), v);
  if (ends && t < sp.nx) {
    const int c = sp.extra(t);
    out[c] = from_f32<T>(g.one(to_f32(row[c]), c, t));
  }
}

// A row without a gradient, whatever it holds.
struct ZeroRow {
  __device__ __forceinline__ float many(float) const { return 0.0f; }
  template <typename V>
  __device__ __forceinline__ void patch(const V&, int, int, V&) const {}
  __device__ __forceinline__ float one(float, int, int) const { return 0.0f; }
};

// Spans of the gradient's rows: one round of four vectors a thread each, so that
// few rows fill the GPU too, and that no span has a round of a few threads left
// (of 1047 vectors as even shares of 6282, it took [4096, 50257] fp16 with 20
// entries 168 us, so 141). Workgroups take a row's spans one after another.
constexpr int kSpan = 4 * kGradThreads;

inline ScorePlan grad_plan(int64_t vocab, int ve) {
  const int64_t nvec = vocab / ve;
  if (nvec < kSpan) return {1, (int)nvec};
  return {(int)((nvec + kSpan - 1) / kSpan), kSpan};
}

// Whether that many bytes pass the 256 MiB last-level cache.
inline bool score_past_cache(int64_t bytes) { return bytes > (int64_t)300 << 20; }

// Argument checks that the row entry points share.
inline int check_score_rows(const char* name, int64_t rows, int64_t vocab, int64_t ld, float temperature,
                            float softcap, int dtype) {
  if (ak_dtype_size(dtype) == 0) return ak_set_error(AK_ERR_UNSUPPORTED, "%s: unsupported dtype code %d", name, dtype);
  if (rows < 0 || vocab <= 0) return ak_set_error(AK_ERR_INVALID_ARG, "%s: bad shape rows=%lld vocab=%lld", name, (long long)rows, (long long)vocab);
  if (vocab > kScoreVocab) return ak_set_error(AK_ERR_UNSUPPORTED, "%s: vocab=%lld is over %lld", name, (long long)vocab, (long long)kScoreVocab);
  if (ld < vocab) return ak_set_error(AK_ERR_INVALID_ARG, "%s: row pitch smaller than vocab", name);
  if (!ak_extent_ok(rows, ld, vocab, ak_dtype_size(dtype)))
    return ak_set_error(AK_ERR_INVALID_ARG, "%s: rows=%lld x pitch exceed 64-bit addressing", name, (long long)rows);
  if (!(temperature >= 1e-18f && temperature <= 1e18f))  // its square is a float, too
    return ak_set_error(AK_ERR_INVALID_ARG, "%s: temperature must be between 1e-18 and 1e18", name);
  // the cap's tanh is within 2^-22 of 1: of a larger cap that is more than the logits' own rounding
  if (!(softcap == 0.0f || (softcap >= 1e-3f && softcap <= 1e4f)))
    return ak_set_error(AK_ERR_INVALID_ARG, "%s: softcap must be 0 or between 1e-3 and 1e4", name);
  // the scores are off by that over the temperature: a quarter there, and further on
  // an element's may pass the row's maximum by more than 2^t holds
  if (softcap > temperature * 0x1p20f)
    return ak_set_error(AK_ERR_INVALID_ARG, "%s: softcap must be at most 2^20 temperatures", name);
  return AK_OK;
}

}  // namespace ak
