// Log probabilities of given tokens, with the entropy and the top alternatives
// of each row of logits, for gfx950.
//
//   y    = softcap > 0 ? softcap * tanh(x / softcap) : x
//   p    = softmax(y / temperature)
//   logp = ln p[token],  H = -sum p ln p,  the top_k largest ln p and their columns
// and backward, with g and e the gradients of logp and H:
//   dx_v = (g ([v == token] - p_v) - e p_v (ln p_v + H)) (1 - tanh^2) / temperature.
//
// HBM-bound: the forward reads the logits once (score_rows.h; of many rows, not
// those of an ignored token), the backward
// reads them once and writes the gradient once. Measured (a copy of 1 GiB here:
// 5.1 TB/s): [8192, 50304] bf16 forward 152 to 160 us, 5.2 TB/s and more, 116 to
// 122 with a quarter of the rows ignored, 136 to 143 for the entropy alone (no
// token's logit to fetch); [4096, 50257] bf16, a quarter ignored, forward 65 us,
// forward and backward 196, 5.2 TB/s over the three passes; [8, 50257] with 20
// alternatives, a decode step, 12 us, two kernels of 3.8 and 9.7 us in a trace.
//
// Alternatives. The first kernel, which has the logits in registers, also
// writes the maximum of each group of consecutive logits (128 bytes of the row
// as a rule: 8 vectors, joined over 8 lanes). The row's top_k largest logits lie
// in the top_k groups of the largest maxima, and in the few logits around the
// row's vectors: each of those groups has a logit at or above the top_k-th
// maximum, and where maxima are equal the groups of lower columns have the
// lower columns. So a second kernel, one wave a row, bisects for the top_k-th
// maximum, reads those groups again (one line each), gathers what passes the
// maximum, and as many logits equal to it as are still wanted, in the order of
// their columns, and places each by counting the larger ones. Keys hold a
// logit's place among the numbers above the complement of its column, so they
// are unique and the result depends on neither the gathering's order nor the
// row's split. -0 equals +0; NaN comes first. Rows with NaN, and rows of which
// more logits pass the bound than LDS holds, are bisected whole (exact_top).
// [4096, 32768] bf16 with 64 alternatives: 49 us for the first kernel, with the
// maxima, and 24 us for the second, 10 of them for lines that the first has
// read already. (With the search, the gathering and the placing in the first kernel, [4096,
// 32768] bf16 with 64 alternatives took 78 to 90 us, where the statistics alone
// take 48: the phases between its barriers left too few loads in flight.)
#include <type_traits>

#include "score_rows.h"

namespace ak {
namespace {

typedef unsigned long long u64;
typedef u64 u64x2 __attribute__((ext_vector_type(2)));

// Places of floats among the numbers, as unsigned integers; NaN first.
__device__ __forceinline__ uint32_t place_of(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
  return (int32_t)u < 0 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float float_at(uint32_t place) {
  return __builtin_bit_cast(float, (int32_t)place < 0 ? place & 0x7FFFFFFFu : ~place);
}
__device__ __forceinline__ u64 key_of(float x, int col) { return (u64)place_of(x) << 32 | (uint32_t)~col; }
__device__ __forceinline__ int key_col(u64 key) { return (int)~(uint32_t)key; }
__device__ __forceinline__ float key_logit(u64 key) { return float_at((uint32_t)(key >> 32)); }

struct LogprobArgs {
  const int64_t* tokens;  // nullable
  float* logprobs;        // with tokens
  float* entropy;         // nullable
  f32x4_t* stats;         // nullable: (m, log2 s, H, -) for the backward
  float* top_logprobs;    // with top > 0
  int64_t* top_ids;
  f32x4_t* part;          // segs > 1 or top > 0: (m, s, u, -) of each segment
  float* maxima;          // top > 0: [rows, groups] maxima of 2^shift vectors each
  int top, vocab, groups, shift;
  // Whether rows of an ignored token are left unread. The token is then waited for
  // before the row: [8192, 50304] bf16 152 to 156 us (154 to 157 without), a quarter
  // of it ignored 116 to 119 (150 to 154), [4096, 50257] 82 to 85 (81 to 84) and 65
  // (81), [2000, 50257] fp32 68 (66) and 54 (66). Few rows, which wait for latency
  // alone, are read.
  bool skip;
};

// The row's results but the alternatives, by one thread.
template <bool CAP>
__device__ __forceinline__ void finish_row(const ScoreParams& p, const LogprobArgs& a, int64_t row, const RowStats& st,
                                           int64_t tok, float x_tok) {
  const float l2 = log2_sum(st);
  float h = row_entropy(st);
  if (a.stats) a.stats[row] = f32x4_t{st.m, l2, h, 0.0f};
  if (a.tokens) {
    float lp;
    if (tok == p.ignore_index) {
      lp = 0.0f;
      h = 0.0f;
    } else if (tok < 0 || tok >= a.vocab) {
      lp = NAN;
    } else {
      lp = log_prob(p, score<CAP>(p, x_tok), st.m, l2);
    }
    a.logprobs[row] = lp;
  }
  if (a.entropy) a.entropy[row] = h;
}

// Alternative r of a row.
template <bool CAP>
__device__ __forceinline__ void store_top(const ScoreParams& p, const LogprobArgs& a, int64_t row, int r, u64 key,
                                          const RowStats& st) {
  const float x = key_logit(key);
  a.top_logprobs[row * a.top + r] = log_prob(p, score<CAP>(p, x), st.m, log2_sum(st));
  a.top_ids[row * a.top + r] = key_col(key);
}

// One workgroup per segment (units by grid stride; the loop bound is uniform).
// SHIFT: kHere where the results are formed here, kPart where they are the
// join's to form, or what 2^SHIFT vectors the groups of alternatives have.
constexpr int kHere = -2, kPart = -1;

template <typename T, int VPT, int TPR, bool CAP, int SHIFT>
__global__ void __launch_bounds__(TPR, AK_SEGMENT_WAVES(VPT))
logprob_segment_kernel(const T* __restrict__ logits, int64_t rows, int64_t ld, int segs, int span, ScoreParams p,
                       LogprobArgs a) {
  constexpr int W = TPR / 64;
  constexpr bool PART = SHIFT != kHere;
  __shared__ float part_m[W], part_s[W], part_u[W];
  for (int64_t unit = blockIdx.x; unit < rows * segs; unit += gridDim.x) {
    const int64_t row = segs == 1 ? unit : unit / segs;
    const int seg = segs == 1 ? 0 : (int)(unit - row * segs);
    const T* x = logits + row * ld;
    int64_t tok = p.ignore_index;
    float x_tok = 0.0f;
    if (SHIFT < 0 && a.tokens && (!PART || a.skip)) {
      tok = a.tokens[row];
      if (a.skip && tok == p.ignore_index) {  // (the whole workgroup) 0 whatever the row holds
        if (threadIdx.x == 0) {
          if (PART) a.part[unit] = f32x4_t{-INFINITY, 0.0f, 0.0f, 0.0f};
          else finish_row<CAP>(p, a, row, RowStats{-INFINITY, 0.0f, 0.0f}, tok, 0.0f);
        }
        continue;
      }
      if (!PART && threadIdx.x == 0 && tok != p.ignore_index && tok >= 0 && tok < a.vocab) x_tok = to_f32(x[tok]);
    }
    Segment<T, VPT, TPR> sg(x, a.vocab, seg, span);
    float m, group[Segment<T, VPT, TPR>::template kStored<(SHIFT > 0 ? SHIFT : 0)>] = {};
    float* const maxima = SHIFT >= 0 ? a.maxima + row * a.groups + seg * (span >> (SHIFT > 0 ? SHIFT : 0)) : nullptr;
    if constexpr (SHIFT >= 0) m = sg.template largest_of_groups<SHIFT>(maxima, group);
    else m = sg.largest();
    m = wave_max(m);
    if ((threadIdx.x & 63) == 0) part_m[threadIdx.x / 64] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) m = fmaxf(m, part_m[i]);
    RowStats st;
    st.m = CAP ? score<CAP>(p, m) : m;
    sg.template sums<CAP, true>(p, st.m, st.s, st.u);
    st.s = wave_sum(st.s);
    st.u = wave_sum(st.u);
    if ((threadIdx.x & 63) == 0) {
      part_s[threadIdx.x / 64] = st.s;
      part_u[threadIdx.x / 64] = st.u;
    }
    __syncthreads();  // part_m has been read by all, so the next unit may write it
    if (threadIdx.x == 0) {
      st.s = part_s[0];
      st.u = part_u[0];
#pragma unroll
      for (int i = 1; i < W; ++i) {
        st.s += part_s[i];
        st.u += part_u[i];
      }
      if (PART) a.part[unit] = f32x4_t{st.m, st.s, st.u, 0.0f};
      else finish_row<CAP>(p, a, row, st, tok, x_tok);
    }
    __syncthreads();  // part_s / part_u are rewritten for the workgroup's next unit
    // (behind the barriers, which would wait for the store)
    if constexpr (SHIFT > 0) sg.template store_groups<SHIFT>(maxima, group);
  }
}

// A row's statistics from its segments, by one wave, in a fixed order.
__device__ __forceinline__ RowStats join_row(const ScoreParams& p, const f32x4_t* part, int segs) {
  RowStats st{-INFINITY, 0.0f, 0.0f};
  if (segs == 1) {
    const f32x4_t q = part[0];
    return RowStats{q[0], q[1], q[2]};
  }
  for (int i = threadIdx.x & 63; i < segs; i += 64) {
    const f32x4_t q = part[i];
    st = join_stats(p, st, RowStats{q[0], q[1], q[2]});
  }
  return wave_join(p, st);
}

// Rows without alternatives from their segments, one wave a row.
template <typename T, bool CAP>
__global__ void __launch_bounds__(64)
logprob_join_kernel(const T* __restrict__ logits, int64_t row0, int64_t ld, int segs, ScoreParams p, LogprobArgs a) {
  const int64_t row = row0 + blockIdx.x;
  int64_t tok = p.ignore_index;
  float x_tok = 0.0f;
  if (threadIdx.x == 0 && a.tokens) {
    tok = a.tokens[row];
    if (tok != p.ignore_index && tok >= 0 && tok < a.vocab) x_tok = to_f32(logits[row * ld + tok]);
  }
  const RowStats st = join_row(p, a.part + row * segs, segs);
  if (threadIdx.x == 0) finish_row<CAP>(p, a, row, st, tok, x_tok);
}

// The bits of a place that tell logits of type T apart.
template <typename T>
constexpr uint32_t kPlaceBits = std::is_same<T, float>::value ? 0xFFFFFFFFu : std::is_same<T, f16>::value ? 0xFFFFE000u : 0xFFFF0000u;

// How many of these lanes are below the calling one.
__device__ __forceinline__ int lanes_before(u64 lanes) {
  return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, 0));
}

// What one row's alternatives are chosen from.
struct Groups {
  const uint16_t* list;  // the chosen groups, ascending
  int n, shift;          // their number; 2^shift vectors a group
};

// Sum of v over the lanes below the calling one, and over all lanes.
__device__ __forceinline__ int lanes_sum_before(int v, int& all) {
  int c = v;  // inclusive: within rows of 16 lanes, then across them
  c += __builtin_amdgcn_update_dpp(0, c, 0x111, 0xF, 0xF, false);  // row_shr 1
  c += __builtin_amdgcn_update_dpp(0, c, 0x112, 0xF, 0xF, false);  // row_shr 2
  c += __builtin_amdgcn_update_dpp(0, c, 0x114, 0xF, 0xF, false);  // row_shr 4
  c += __builtin_amdgcn_update_dpp(0, c, 0x118, 0xF, 0xF, false);  // row_shr 8
  c += __builtin_amdgcn_update_dpp(0, c, 0x142, 0xA, 0xF, false);  // row_bcast 15, into rows 1 and 3
  c += __builtin_amdgcn_update_dpp(0, c, 0x143, 0xC, 0xF, false);  // row_bcast 31, into rows 2 and 3
  all = __builtin_amdgcn_readlane(c, 63);
  return c - v;
}

// Gathers the keys of the logits of the chosen groups that `passes` takes, in
// any order; where a wave has the row alone, the loads of eight vectors a thread
// are in flight before the first is used. Reached by whole waves; what `count` passes CAND by is left out.
template <typename T, int TT, int CAND, typename F>
__device__ __forceinline__ void gather_chosen(const T* __restrict__ row, const RowSplit<T>& sp, const Groups& g, u64* cand,
                                              int* count, F passes) {
  constexpr int VE = Vec16<T>::VE, U = TT > 64 ? 2 : 8;
  const int total = g.n << g.shift, lane = threadIdx.x & 63;
  for (int i0 = threadIdx.x - lane; i0 < total; i0 += U * TT) {
    Vec16<T> q[U];
    int col[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + lane + u * TT;
      const int v = i < total ? (g.list[i >> g.shift] << g.shift) + (i & ((1 << g.shift) - 1)) : sp.nvec;
      col[u] = v < sp.nvec ? sp.head + v * VE : -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (col[u] >= 0) q[u] = load16_any(row + col[u]);
    uint32_t mask[U];  // bit e: element e of vector u passes
    int mine = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint32_t m = 0;
#pragma unroll
      for (int e = 0; e < VE; ++e) m |= passes(to_f32(q[u].e[e])) ? 1u << e : 0u;
      mask[u] = col[u] >= 0 ? m : 0u;
      mine += __popc(mask[u]);
    }
    int all, to = lanes_sum_before(mine, all);
    if (all == 0) continue;
    int base = 0;
    if (lane == 0) base = atomicAdd(count, all);
    to += __builtin_amdgcn_readfirstlane(base);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (mask[u]) {
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          if (mask[u] >> e & 1) {
            if (to < CAND) cand[to] = key_of(to_f32(q[u].e[e]), col[u] + e);
            ++to;
          }
        }
      }
    }
  }
}

// The keys of a row's `top` largest logits, gathered in any order: a search by
// two bits at a time for the top-th largest place, then for the column up to
// which logits of that place belong to the top, the row read again for each
// step. For rows with NaN, and rows of which too many logits pass the bound.
// Reached by the whole workgroup; part: 64 bits a wave.
template <typename T, int TT>
__device__ int exact_top(const T* __restrict__ row, int vocab, int top, u64* cand, int* count, u64* part) {
  const int t = threadIdx.x;
  auto each = [&](auto f) {
#pragma unroll 4
    for (int i = t; i < vocab; i += TT) f(place_of(to_f32(row[i])), i);
  };
  // which(place, column): up to three counts of 21 bits
  auto total = [&](auto which) {
    u64 c = 0;
    each([&](uint32_t q, int col) { c += which(q, col); });
    for (int off = 32; off >= 1; off >>= 1) c += __shfl_xor(c, off, 64);
    __syncthreads();  // the last total has been read
    if ((t & 63) == 0) part[t / 64] = c;
    __syncthreads();
    c = 0;
    for (int i = 0; i < TT / 64; ++i) c += part[i];
    return c;
  };
  auto of = [](u64 c, int j) { return (int)(c >> (21 * (j - 1))) & 0x1FFFFF; };
  auto three = [](bool a, bool b, bool c) { return (u64)a | (u64)b << 21 | (u64)c << 42; };
  uint32_t place = 0;
#pragma unroll 1
  for (int sh = 30; sh >= 0; sh -= 2) {
    const uint32_t at = 1u << sh;
    const u64 c = total([&](uint32_t q, int) { return three(q >= place + at, q >= place + 2 * at, q >= place + 3 * at); });
    int j = 3;
    while (j > 0 && of(c, j) < top) --j;
    place += j * at;
  }
  const int need = top - of(total([&](uint32_t q, int) { return three(q > place, false, false); }), 1);
  int last = 0;  // the column of the need-th logit of that place
#pragma unroll 1
  for (int sh = 18; sh >= 0; sh -= 2) {
    const int at = 1 << sh;
    const u64 c = total([&](uint32_t q, int col) {
      return q == place ? three(col < last + at, col < last + 2 * at, col < last + 3 * at) : 0;
    });
    int j = 3;
    while (j > 0 && of(c, j) >= need) --j;
    last += j * at;
  }
  __syncthreads();
  if (t == 0) *count = 0;
  __syncthreads();
  each([&](uint32_t q, int col) {
    if (q > place || (q == place && col <= last)) cand[atomicAdd(count, 1)] = (u64)q << 32 | (uint32_t)~col;
  });
  __syncthreads();
  return *count;
}

// Groups that may be chosen beyond top: the search ends some bits earlier.
constexpr int kSpare = 16;

// A row's results from its segments' statistics and its groups' maxima. TT
// threads a row: one wave where there are rows enough, four where there are few.
// MAXG, CAND: room for the maxima and for the keys of what passes the bound.
template <typename T, bool CAP, int TT, int MAXG, int CAND>
__global__ void __launch_bounds__(TT)
logprob_top_kernel(const T* __restrict__ logits, int64_t row0, int64_t ld, int segs, ScoreParams p, LogprobArgs a) {
  constexpr int VE = Vec16<T>::VE;
  static_assert(MAXG <= 65536 && MAXG % 64 == 0 && CAND >= kMaxTop, "groups in 16 bits, whole rounds");
  __shared__ __attribute__((aligned(16))) u64 cand[CAND + 2];
  __shared__ uint16_t list[kMaxTop + kSpare];
  __shared__ u64 totals[TT / 64];
  __shared__ RowStats whole;
  __shared__ uint32_t bound;
  __shared__ int count, chosen;
  const int64_t row = row0 + blockIdx.x;
  const T* x = logits + row * ld;
  const RowSplit<T> sp(x, a.vocab);
  const int t = threadIdx.x, lane = t & 63;
  // (with an address off the 16-byte grid a row may have one vector less than its groups hold)
  const int groups = (sp.nvec + (1 << a.shift) - 1) >> a.shift;
  const uint32_t least_place = place_of(-INFINITY) & kPlaceBits<T>;
  constexpr int kStatsWave = TT > 64 ? 64 : 0;  // the threads that fold the statistics, meanwhile where there are others
  if (t < 64) {
    constexpr int PER = MAXG / 64;
    uint32_t q[PER];  // places, 0 behind the last group (no logit has place 0)
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = i * 64 + lane;
      q[i] = at < groups ? __builtin_bit_cast(uint32_t, a.maxima[row * a.groups + at]) : 0u;
    }
    uint32_t high = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      q[i] = i * 64 + lane < groups ? place_of(__builtin_bit_cast(float, q[i])) & kPlaceBits<T> : 0u;
      high = max(high, q[i]);
    }
    auto number = [&](auto which) {
      int c = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) c += __popcll(__ballot(which(q[i])));
      return c;
    };
    uint32_t b = least_place;
    bool all = false;  // whether few more than top maxima reach b: all those are chosen then
    if (groups > a.top) {
      for (int off = 32; off >= 1; off >>= 1) high = max(high, (uint32_t)__shfl_xor((int)high, off, 64));
      b = 0;
      // the top-th largest maximum, bit by bit (those above the largest's first are 0 in every place)
      for (int bit = 31 - __builtin_clz(high | 1u); bit >= __builtin_ctz(kPlaceBits<T>) && !all; --bit) {
        const uint32_t at = b | 1u << bit;
        const int c = number([&](uint32_t v) { return v >= at; });
        if (c >= a.top) b = at;
        all = c >= a.top && c <= a.top + kSpare;
      }
      b = max(b, least_place);  // (every maximum reaches it: below it are no numbers)
    }
    // the chosen groups, ascending: those that reach b, or those above it and as
    // many of those at it as are wanted
    int left = all ? MAXG : a.top - number([&](uint32_t v) { return v > b; }), to = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const u64 ties = __ballot(q[i] == b);
      const bool take = q[i] > b || (q[i] == b && lanes_before(ties) < left);
      const u64 taken = __ballot(take);
      if (take) list[to + lanes_before(taken)] = (uint16_t)(i * 64 + lane);
      to += __popcll(taken);
      left = max(0, left - (int)__popcll(ties));
    }
    if (lane == 0) {
      chosen = to;
      bound = b;
      count = 0;
    }
  }
  if (t >= kStatsWave && t < kStatsWave + 64) {
    const int64_t tok = lane == 0 && a.tokens ? a.tokens[row] : p.ignore_index;
    float x_tok = 0.0f;
    if (tok != p.ignore_index && tok >= 0 && tok < a.vocab) x_tok = to_f32(x[tok]);
    const RowStats st = join_row(p, a.part + row * segs, segs);
    if (lane == 0) {
      whole = st;
      finish_row<CAP>(p, a, row, st, tok, x_tok);
    }
  }
  __syncthreads();
  const Groups g{list, chosen, a.shift};
  const float least = float_at(bound < 0x80000000u ? bound | ~kPlaceBits<T> : bound);  // (a negative number's low bits are set)
  // what reaches the bound in the chosen groups, or what passes it
  bool above = false;
  auto passes = [&](float v) { return above ? v > least : v >= least; };
  auto gather = [&]() {
    gather_chosen<T, TT, CAND>(x, sp, g, cand, &count, passes);
    if (t < sp.nx && passes(to_f32(x[sp.extra(t)]))) {
      const int at = atomicAdd(&count, 1);
      if (at < CAND) cand[at] = key_of(to_f32(x[sp.extra(t)]), sp.extra(t));
    }
    __syncthreads();
  };
  gather();
  const RowStats st = whole;
  int n = count;
  const bool nan = st.s != st.s;
  if (n > CAND && !nan) {  // uniform, as below
    // many logits equal to the bound: those above it, and of the equal ones as
    // many as are still wanted, by column: those before the row's vectors,
    // those of the chosen groups, those behind
    __syncthreads();
    if (t == 0) count = 0;
    above = true;
    __syncthreads();
    gather();
    if (t < 64 && count < a.top) {
      int at = count;
      auto in_order = [&](bool equal, int col) {
        const u64 lanes = __ballot(equal);
        const int i = at + lanes_before(lanes);
        if (equal && i < a.top) cand[i] = key_of(least, col);
        at = min(a.top, at + (int)__popcll(lanes));
      };
      const bool ex = t < sp.nx && to_f32(x[sp.extra(t)]) == least;
      in_order(ex && t < sp.head, t);
      const int total = g.n << g.shift;
      for (int i0 = 0; i0 < total && at < a.top; i0 += 64) {
        const int i = i0 + lane, v = i < total ? (g.list[i >> g.shift] << g.shift) + (i & ((1 << g.shift) - 1)) : sp.nvec;
        uint32_t equal = 0;  // bit e: element e of this lane's vector
        if (v < sp.nvec) {
          const Vec16<T> q = load16_any(x + sp.head + v * VE);
#pragma unroll
          for (int e = 0; e < VE; ++e) equal |= (uint32_t)(to_f32(q.e[e]) == least) << e;
        }
        // lanes are in the order of columns, a lane's elements follow each other
        int before = 0, sum = 0;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const u64 lanes = __ballot(equal >> e & 1);
          before += lanes_before(lanes);
          sum += __popcll(lanes);
        }
        int k = at + before;
        for (uint32_t rest = equal; rest && k < a.top; rest &= rest - 1, ++k)
          cand[k] = key_of(least, sp.head + v * VE + __builtin_ctz(rest));
        at = min(a.top, at + sum);
      }
      in_order(ex && t >= sp.head, sp.extra(t));
      if (t == 0) count = at;
    }
    __syncthreads();
    n = count;
  }
  if (n > CAND || nan) n = exact_top<T, TT>(x, a.vocab, a.top, cand, &count, totals);
  if (t < 2) cand[n + t] = 0;
  __syncthreads();
  for (int c = t; c < n; c += TT) {
    const u64 key = cand[c];
    int r = 0;
#pragma unroll 4
    for (int i = 0; i < n; i += 2) {
      const u64x2 two = *reinterpret_cast<const u64x2*>(cand + i);
      r += (two[0] > key) + (two[1] > key);
    }
    if (r < a.top) store_top<CAP>(p, a, row, r, key, st);
  }
}

// -(g + e (ln p + H)) = c0 + c1 log2 p, and g for the given token beside it.
template <typename T, bool CAP>
struct LogprobRow {
  const ScoreParams& p;
  float m, l2, c0, c1, g;
  int token;
  __device__ __forceinline__ float many(float x) const {
    float slope;
    const float y = score_and_slope<T, CAP>(p, x, slope);
    const float lp = (y - m) * p.c2 - l2;
    // p is 0 from -150 on, and log2 p may be -inf there
    return __builtin_amdgcn_exp2f(lp) * fmaf(c1, fmaxf(lp, -1000.0f), c0) * slope;
  }
  __device__ __forceinline__ float one(float x, int col, int) const {
    float slope;
    score_and_slope<T, CAP>(p, x, slope);
    return col == token ? fmaf(g, slope, many(x)) : many(x);
  }
  __device__ __forceinline__ void patch(const Vec16<T>& x, int col, int, Vec16<T>& o) const {
    if ((unsigned)(token - col) >= (unsigned)Vec16<T>::VE) return;
#pragma unroll
    for (int e = 0; e < Vec16<T>::VE; ++e)
      if (col + e == token) o.e[e] = from_f32<T>(one(to_f32(x.e[e]), col + e, 0));
  }
};

// The gradient from the forward's statistics; a workgroup takes `span` vectors
// of a row.
template <typename T, bool CAP, bool NT, int U>
__global__ void __launch_bounds__(kGradThreads)
logprob_grad_kernel(const T* __restrict__ logits, const int64_t* __restrict__ tokens, const f32x4_t* __restrict__ stats,
                    const float* __restrict__ g_logprobs, const float* __restrict__ g_entropy, T* __restrict__ grad,
                    int64_t rows, int vocab, int64_t ld, int64_t ld_g, int spans, int span, ScoreParams p) {
  for (int64_t unit = blockIdx.x; unit < rows * spans; unit += gridDim.x) {
    const int64_t row = unit / spans;
    const int v0 = (int)(unit - row * spans) * span, v1 = v0 + span;
    const bool ends = v0 == 0;
    const T* x = logits + row * ld;
    T* gx = grad + row * ld_g;
    const f32x4_t st = stats[row];
    const int64_t tok = tokens ? tokens[row] : -1;
    const bool ignored = tokens && tok == p.ignore_index;
    const bool bad = tokens && !ignored && (tok < 0 || tok >= vocab);
    const bool empty = st[0] == -INFINITY && st[1] == 0.0f;
    if (ignored || empty) {
      map_row<T, NT, 1>(x, gx, vocab, v0, v1, ends, ZeroRow());
      continue;
    }
    const float g = bad ? NAN : (tokens && g_logprobs ? g_logprobs[row] : 0.0f);
    const float e = g_entropy ? g_entropy[row] : 0.0f;
    const LogprobRow<T, CAP> f{p, st[0], st[1], -fmaf(e, st[2], g), -e * kLn2, g, tokens && !bad ? (int)tok : -1};
    map_row<T, NT, U>(x, gx, vocab, v0, v1, ends, f);
  }
}

// The groups of a row whose maxima are kept: 64 vectors where that leaves
// twice the alternatives and 256 of them, else 8 (one line) where that leaves
// twice the alternatives, else single vectors. Up to kMaxGroups.
constexpr int kMaxGroups = 4096;

int group_shift(int64_t nvec, int top) {
  if (nvec / 64 >= std::max(2 * top, 256)) return 6;
  return nvec / 8 >= 2 * top ? 3 : 0;
}

struct Workspace {
  int shift, groups;
  size_t part, maxima, total;
};

Workspace workspace(int64_t rows, int64_t vocab, int ve, const ScorePlan& pl, int top) {
  auto up = [](size_t v) { return (v + 255) & ~(size_t)255; };
  Workspace w{0, 0, 0, 0, 0};
  if ((pl.segs == 1 && top == 0) || rows <= 0) return w;
  w.maxima = w.total = up((size_t)rows * pl.segs * sizeof(f32x4_t));
  if (top > 0) {
    const int64_t nvec = std::max<int64_t>(1, vocab / ve);
    w.shift = group_shift(nvec, top);
    w.groups = (int)((nvec + (1 << w.shift) - 1) >> w.shift);
    w.total += up((size_t)rows * w.groups * sizeof(float));
  }
  return w;
}

template <typename T, bool CAP>
void launch_fwd(const void* logits, int64_t rows, int64_t ld, const ScorePlan& pl, const ScoreParams& p,
                const LogprobArgs& a, hipStream_t s) {
  const T* x = static_cast<const T*>(logits);
  const dim3 grid(row_grid(rows * pl.segs));
  auto segments = [&](auto shift) {
    constexpr int SHIFT = decltype(shift)::value;
#define GO(VPT, TPR) logprob_segment_kernel<T, VPT, TPR, CAP, SHIFT><<<grid, dim3(TPR), 0, s>>>(x, rows, ld, pl.segs, pl.span, p, a)
    AK_SEGMENT_DISPATCH(pl.span, GO);
#undef GO
  };
  if (!a.part) segments(std::integral_constant<int, kHere>());
  else if (a.top == 0) segments(std::integral_constant<int, kPart>());
  else if (a.shift == 0) segments(std::integral_constant<int, 0>());
  else if (a.shift == 3) segments(std::integral_constant<int, 3>());
  else segments(std::integral_constant<int, 6>());
  if (!a.part) return;
  // One wave a row where every CU has two, four waves for fewer rows and the
  // widest. Room for the keys that reach the bound: about 1.4 top of twice top
  // groups, fewer of more; where a row has less than twice top groups (of single
  // vectors then) all of its logits may.
  const bool few = rows < 512;
  for (int64_t row0 = 0; row0 < rows; row0 += kMaxRowGrid) {
    const dim3 each(row_grid(rows - row0));
#define TOP(TT, MAXG, CAND) logprob_top_kernel<T, CAP, TT, MAXG, CAND><<<each, dim3(TT), 0, s>>>(x, row0, ld, pl.segs, p, a)
    if (a.top == 0) logprob_join_kernel<T, CAP><<<each, dim3(64), 0, s>>>(x, row0, ld, pl.segs, p, a);
    else if (a.groups < 2 * a.top || a.groups > 2048) TOP(256, kMaxGroups, 2048);
    else if ((a.groups > 1024 || a.top > 128) && few) TOP(256, 2048, 1024);
    else if (a.groups > 1024 || a.top > 128) TOP(64, 2048, 1024);
    else if (few) TOP(256, 1024, 512);
    else if (a.groups > 512) TOP(64, 1024, 512);
    else TOP(64, 512, 512);
#undef TOP
  }
}

template <typename T, bool CAP>
void launch_bwd(const void* logits, const int64_t* tokens, const float* stats, const float* gl, const float* ge,
                void* grad, int64_t rows, int vocab, int64_t ld, int64_t ld_g, const ScoreParams& p, hipStream_t s) {
  constexpr int VE = Vec16<T>::VE;
  const ScorePlan pl = grad_plan(vocab, VE);
  const dim3 grid(row_grid(rows * pl.segs)), block(kGradThreads);
  const T* x = static_cast<const T*>(logits);
  T* g = static_cast<T*>(grad);
  const f32x4_t* st = reinterpret_cast<const f32x4_t*>(stats);
  if (vocab / VE < 4 * kGradThreads)
    logprob_grad_kernel<T, CAP, false, 1><<<grid, block, 0, s>>>(x, tokens, st, gl, ge, g, rows, vocab, ld, ld_g, pl.segs, pl.span, p);
  else if (score_past_cache(2 * rows * vocab * (int64_t)sizeof(T)))
    logprob_grad_kernel<T, CAP, true, 4><<<grid, block, 0, s>>>(x, tokens, st, gl, ge, g, rows, vocab, ld, ld_g, pl.segs, pl.span, p);
  else
    logprob_grad_kernel<T, CAP, false, 4><<<grid, block, 0, s>>>(x, tokens, st, gl, ge, g, rows, vocab, ld, ld_g, pl.segs, pl.span, p);
}

}  // namespace
}  // namespace ak

extern "C" size_t ak_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int top_k, int dtype) {
  const int esz = ak_dtype_size(dtype);
  if (rows <= 0 || vocab <= 0 || vocab > ak::kScoreVocab || top_k < 0 || top_k > ak::kMaxTop || esz == 0) return 0;
  return ak::workspace(rows, vocab, 16 / esz, ak::score_plan(rows, vocab, 16 / esz), top_k).total;
}

extern "C" int ak_token_logprobs_fwd(const void* logits, const int64_t* tokens, float* logprobs, float* entropy,
                                     float* stats, float* top_logprobs, int64_t* top_ids, void* workspace,
                                     size_t workspace_bytes, int64_t rows, int64_t vocab, int64_t ld_logits,
                                     int top_k, float temperature, float softcap, int64_t ignore_index, int dtype,
                                     void* stream) {
  const char* name = "ak_token_logprobs_fwd";
  int rc = ak::check_score_rows(name, rows, vocab, ld_logits, temperature, softcap, dtype);
  if (rc) return rc;
  if (top_k < 0 || top_k > ak::kMaxTop || top_k > vocab)
    return ak_set_error(AK_ERR_INVALID_ARG, "%s: top_k=%d must be between 0 and min(%d, vocab)", name, top_k, ak::kMaxTop);
  if (rows == 0) return AK_OK;
  if (!logits || (tokens && !logprobs) || (top_k > 0 && (!top_logprobs || !top_ids)))
    return ak_set_error(AK_ERR_INVALID_ARG, "%s: null pointer", name);
  if (stats && !ak::aligned16(stats)) return ak_set_error(AK_ERR_INVALID_ARG, "%s: stats must be 16-byte aligned", name);
  const int ve = 16 / ak_dtype_size(dtype);
  const ak::ScorePlan pl = ak::score_plan(rows, vocab, ve);
  const ak::Workspace w = ak::workspace(rows, vocab, ve, pl, top_k);
  if (workspace_bytes < w.total || (w.total && (!workspace || !ak::aligned16(workspace))))
    return ak_set_error(AK_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed (16-byte aligned)", name, workspace_bytes, w.total);
  char* ws = static_cast<char*>(workspace);
  const ak::LogprobArgs a{tokens, logprobs, entropy, reinterpret_cast<ak::f32x4_t*>(stats), top_logprobs, top_ids,
                          w.total ? reinterpret_cast<ak::f32x4_t*>(ws) : nullptr, reinterpret_cast<float*>(ws + w.maxima),
                          top_k, (int)vocab, w.groups, w.shift, rows >= 256 && top_k == 0};
  const ak::ScoreParams p = ak::score_params(temperature, softcap, ignore_index);
  hipStream_t s = ak_stream(stream);
  auto go = [&](auto t) {
    using T = decltype(t);
    if (softcap > 0.0f) ak::launch_fwd<T, true>(logits, rows, ld_logits, pl, p, a, s);
    else ak::launch_fwd<T, false>(logits, rows, ld_logits, pl, p, a, s);
  };
  if (dtype == AK_DTYPE_F32) go(float());
  else if (dtype == AK_DTYPE_F16) go(ak::f16());
  else go(ak::bf16());
  return ak_check_launch(name);
}

extern "C" int ak_token_logprobs_bwd(const void* logits, const int64_t* tokens, const float* stats,
                                     const float* grad_logprobs, const float* grad_entropy, void* grad_logits,
                                     int64_t rows, int64_t vocab, int64_t ld_logits, int64_t ld_grad,
                                     float temperature, float softcap, int64_t ignore_index, int dtype,
                                     void* stream) {
  const char* name = "ak_token_logprobs_bwd";
  int rc = ak::check_score_rows(name, rows, vocab, std::min(ld_logits, ld_grad), temperature, softcap, dtype);
  if (!rc) rc = ak::check_score_rows(name, rows, vocab, std::max(ld_logits, ld_grad), temperature, softcap, dtype);
  if (rc) return rc;
  if (rows == 0) return AK_OK;
  if (!logits || !stats || !grad_logits) return ak_set_error(AK_ERR_INVALID_ARG, "%s: null pointer", name);
  if (!ak::aligned16(stats)) return ak_set_error(AK_ERR_INVALID_ARG, "%s: stats must be 16-byte aligned", name);
  const ak::ScoreParams p = ak::score_params(temperature, softcap, ignore_index);
  hipStream_t s = ak_stream(stream);
  auto go = [&](auto t) {
    using T = decltype(t);
    if (softcap > 0.0f) ak::launch_bwd<T, true>(logits, tokens, stats, grad_logprobs, grad_entropy, grad_logits, rows, (int)vocab, ld_logits, ld_grad, p, s);
    else ak::launch_bwd<T, false>(logits, tokens, stats, grad_logprobs, grad_entropy, grad_logits, rows, (int)vocab, ld_logits, ld_grad, p, s);
  };
  if (dtype == AK_DTYPE_F32) go(float());
  else if (dtype == AK_DTYPE_F16) go(ak::f16());
  else go(ak::bf16());
  return ak_check_launch(name);
}
