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
__device__ __forceinline__ void sequence_tokens(const Sequences& s, int b, int& first, int& count) {
  if (s.starts == nullptr) {
    first = b * (int)s.per;
    count = (int)s.per;
    return;
  }
  const int tokens = (int)s.tokens;
  first = min(max(s.starts[b], 0), tokens);
  count = max(min(s.starts[b + 1], tokens) - first, 0);
}

// The sequence of token t (the last b with starts[b] <= t), or -1 where none has
// it. All lanes of the wave search for their own t together: 64 starts at a time
// narrow the lowest lane's sequence down, the others walk on from there (their
// tokens follow it).
__device__ __forceinline__ int sequence_of(const Sequences& s, int t) {
  const int batch = (int)s.batch;
  if (batch == 0) return -1;
  if (s.starts == nullptr) return (uint32_t)t / (uint32_t)s.per;
  const int lane = threadIdx.x & 63;
  const int t0 = __builtin_amdgcn_readfirstlane(t);
  uint32_t lo = 0, n = batch;  // starts[lo] <= t0 (or lo = 0), starts[lo + n] > t0 (or the end)
  while (n > 1) {
    const uint32_t step = (n + 63) / 64, at = lane * step;
    const bool le = at < n && s.starts[lo + at] <= t0;
    const uint64_t hit = __ballot(le);
    const uint32_t last = (hit ? 63 - __builtin_clzll(hit) : 0) * step;
    lo += last;
    n = min(step, n - last);
  }
  int b = (int)lo;
  int first = s.starts[b], next = s.starts[b + 1];
  while (next <= t && b + 1 < batch) {
    ++b;
    first = next;
    next = s.starts[b + 1];
  }
  return first <= t && t < next ? b : -1;
}

// Division by a number of up to 32 bits that a launch knows.
struct Divisor {
  uint32_t d, magic;  // 2^32 / d, rounded down
  Divisor() = default;
  explicit Divisor(int64_t n) : d((uint32_t)n), magic((uint32_t)(n < 2 ? UINT32_MAX : ((uint64_t)1 << 32) / (uint64_t)n)) {}
  __device__ __forceinline__ uint32_t operator()(uint32_t x) const {
    const uint32_t q = __umulhi(x, magic);  // the quotient or one less
    return x - q * d >= d ? q + 1 : q;
  }
};

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
