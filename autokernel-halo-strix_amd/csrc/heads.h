// Shared pieces of the operators on attention heads (rotary positions, head
// norms, the paged cache): sequence search, page lookup.
#pragma once

#include "ak_common.h"

namespace ak {

constexpr int64_t kMaxHeadDim = 2048;

// A batch of sequences with new tokens each: sequence b's are the rows
// [starts[b], starts[b + 1]) of the call's tokens (NULL: `per` tokens each) and
// the last ones of its lengths[b] positions.
struct Sequences {
  const int32_t* starts;
  const int32_t* lengths;
  int64_t batch, tokens, per;
};

// The first new token of sequence b and the number of them, inside the call's
// tokens whatever `starts` holds.
__device__ __forceinline__ void sequence_tokens(const Sequences& s, int64_t b, int64_t& first, int64_t& count) {
  if (s.starts == nullptr) {
    first = b * s.per;
    count = s.per;
    return;
  }
  const int64_t a = s.starts[b], e = s.starts[b + 1];
  first = min(max(a, (int64_t)0), s.tokens);
  count = max(min(e, s.tokens) - first, (int64_t)0);
}

// The sequence of token t (the last b with starts[b] <= t), or -1 where none has
// it. All lanes of the wave search for their own t together: 64 starts at a time
// narrow the lowest lane's sequence down, the others walk on from there (their
// tokens follow it).
__device__ __forceinline__ int64_t sequence_of(const Sequences& s, int64_t t) {
  if (s.batch == 0) return -1;
  if (s.starts == nullptr) return (uint32_t)t / (uint32_t)s.per;
  const int lane = threadIdx.x & 63;
  const int64_t t0 = ((int64_t)__builtin_amdgcn_readfirstlane((int)(t >> 32)) << 32) |
                     (uint32_t)__builtin_amdgcn_readfirstlane((int)t);
  int64_t lo = 0, n = s.batch;  // starts[lo] <= t0 (or lo = 0), starts[lo + n] > t0 (or the end)
  while (n > 1) {
    const int64_t step = (n + 63) / 64;
    const int64_t i = lo + lane * step;
    const bool le = lane * step < n && s.starts[i] <= t0;
    const uint64_t hit = __ballot(le);
    const int last = hit ? 63 - __builtin_clzll(hit) : 0;
    const int64_t nlo = lo + last * step;
    n = min(step, lo + n - nlo);
    lo = nlo;
  }
  int64_t b = lo;
  while (b + 1 < s.batch && s.starts[b + 1] <= t) ++b;
  return s.starts[b] <= t && t < s.starts[b + 1] ? b : -1;
}

// Whether (outer, inner, heads) rows of dim elements at these strides stay
// addressable with signed 64-bit byte offsets.
inline bool extent_ok(int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t n2, int64_t s2, int64_t dim, int esz) {
  if (s0 < 0 || s1 < 0 || s2 < 0) return false;
  const __int128 last = (__int128)(n0 - 1) * s0 + (__int128)(n1 - 1) * s1 + (__int128)(n2 - 1) * s2 + dim;
  return n0 <= 0 || n1 <= 0 || n2 <= 0 || last <= INT64_MAX / esz;
}

// The arguments that every operator on a paged cache checks alike.
inline int check_paged(const char* name, int64_t tokens, int64_t batch, int64_t n_pages, int64_t page_size,
                       int64_t max_pages, int64_t ld_pages, const int32_t* starts, const int32_t* lengths,
                       const int32_t* page_table) {
  if (tokens < 0 || batch < 0 || n_pages < 0 || page_size < 1 || max_pages < 0 || batch > INT32_MAX || tokens > INT32_MAX ||
      n_pages > INT32_MAX || page_size > INT32_MAX || ld_pages < 0 || (batch > 1 && ld_pages < max_pages) ||
      (batch > 1 && ld_pages > INT64_MAX / 8 / batch))
    return ak_set_error(AK_ERR_INVALID_ARG, "%s: bad shape of the batch or the pages", name);
  if (!starts && tokens > 0 && (batch == 0 || tokens % batch))
    return ak_set_error(AK_ERR_INVALID_ARG, "%s: %lld tokens are not the same number for each of %lld sequences", name,
                        (long long)tokens, (long long)batch);
  if (tokens > 0 && batch > 0 && (!lengths || (max_pages > 0 && !page_table)))
    return ak_set_error(AK_ERR_INVALID_ARG, "%s: null pointer", name);
  return AK_OK;
}

}  // namespace ak
