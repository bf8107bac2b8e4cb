// Shared pieces of the kernels of attention over a paged cache.
#pragma once

#include "heads.h"

namespace ak {

constexpr int64_t kMaxAttendDim = 1024;
constexpr float kNegInf = -__builtin_inff();

struct AttendArgs {
  const void *q, *k, *v;
  void* out;
  float* part;
  Sequences seq;
  const int32_t* pages;
  int64_t n_pages, page_size, max_pages, ld_pages;
  int64_t q_st, q_sh, o_st, o_sh;
  int64_t kp, ks, kh, vp, vs, vh;  // cache strides: page, slot, head
  int64_t window;                  // 0: none
  int q_heads, kv_heads, dim, zero_other;
  int splits;
  float scale, softcap;
};

// The keys that a token at `pos` of a sequence may see: [lo, hi).
__device__ __forceinline__ void keys_of(const AttendArgs& a, int64_t length, int64_t pos, int64_t& lo, int64_t& hi) {
  hi = min(pos + 1, min(length, a.max_pages * a.page_size));
  lo = a.window > 0 ? max(pos - a.window + 1, (int64_t)0) : 0;
  if (hi < lo) hi = lo;
}

// The page of key j of sequence b, or -1 where there is none.
__device__ __forceinline__ int64_t page_of(const AttendArgs& a, int64_t b, int64_t j, int64_t& slot) {
  const int64_t i = (uint32_t)j / (uint32_t)a.page_size;
  slot = j - i * a.page_size;
  const int64_t page = a.pages[b * a.ld_pages + i];
  return page >= 0 && page < a.n_pages ? page : -1;
}

// tanh(x) for a cap's product, its error relative to the result (within 4 units of 2^-24): below
// 1 the sixth convergent of Lambert's continued fraction x / (1 + x^2 / (3 + x^2 / (5 + ..))),
// off by 7e-10 of it at 1; from there (1 - e) / (1 + e), e = exp(-2 |x|), whose difference from 1
// has lost what is small (scores within 10 under a cap of 1e4 were off by 1.5e-4). One
// division for both: a reciprocal and a residual step.
__device__ __forceinline__ float cap_tanh(float x) {
  const float a = fabsf(x), t = x * x, e = fast_exp(-2.0f * a);
  const bool small = a < 1.0f;
  const float n = small ? a * fmaf(fmaf(21.0f, t, 1260.0f), t, 10395.0f) : 1.0f - e;
  const float d = small ? fmaf(fmaf(t + 210.0f, t, 4725.0f), t, 10395.0f) : 1.0f + e;
  const float q = __builtin_amdgcn_rcpf(d);
  float r = n * q;
  r = fmaf(fmaf(-d, r, n), q, r);
  return copysignf(r, x);
}

// A row's scores as the running maximum takes them: capped, or the bare products, whose factor
// joins in the exponents (a product that fp32 holds counts as itself whatever the factor).
__device__ __forceinline__ float score_of(const AttendArgs& a, float dot) {
  return a.softcap > 0.0f ? a.softcap * cap_tanh(dot * a.scale / a.softcap) : dot;
}
__device__ __forceinline__ float score_factor(const AttendArgs& a) { return a.softcap > 0.0f ? 1.0f : a.scale; }

// exp(factor (s - m)); beside a maximum of -inf (nothing seen yet, or NaN alone, which the
// maximum passes over) 0 or that NaN.
__device__ __forceinline__ float weight_of(float s, float m, float factor) {
  return m == kNegInf ? (s == s ? 0.0f : s) : fast_exp((s - m) * factor);
}

// The kernels on the matrix cores (paged_attention_tiles.hip): fp16 / bf16 of head
// dims up to 256 in whole 16-byte vectors, fp32 the same.
bool attend_tiles_take(const AttendArgs& a, int dtype);
size_t attend_tiles_workspace_bytes(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim,
                                    int64_t max_keys, int64_t max_chunk, int dtype);
void attend_tiles(const AttendArgs& a, int64_t max_chunk, int dtype, void* workspace, hipStream_t s);

}  // namespace ak
