// Log probabilities of given tokens, with the entropy and the top alternatives
// of each row of logits, for gfx950.
//
//   y    = softcap > 0 ? softcap * tanh(x / softcap) : x
//   p    = softmax(y / temperature)
//   logp = ln p[token],  H = -sum p ln p,  the top_k largest ln p and their columns
// and backward, with g and e the gradients of logp and H:
//   dx_v = (g ([v == token] - p_v) - e p_v (ln p_v + H)) (1 - tanh^2) / temperature.
//
// HBM-bound: the forward reads the logits once (score_rows.h), the backward
// reads them once and writes the gradient once.
//
// Alternatives. Every thread has the largest of the (at most 64) logits it
// holds from the max pass. The top_k-th largest of these group maxima is a
// lower bound of the row's top_k-th logit, since top_k groups reach it; few
// other logits do (for random rows about G ln(G / (G - K)) of them reach the
// bound of G groups: 66 for 64 of 1024). So the threshold comes from one
// wave's search over the maxima while the others form their exponentials, the
// logits that reach it are gathered in LDS, and each finds its place by
// counting the larger ones. Rows of which too many reach the threshold
// (thousands of equal logits) and rows with NaN find the exact bound by
// bisection over the whole segment (exact_top). A key holds the logit's place among the
// numbers above the complement of its column, so keys are unique, equal logits
// go by column and the result depends on neither the gathering's order nor
// the row's split. -0 equals +0; NaN comes first.
#include <type_traits>

#include "score_rows.h"

namespace ak {
namespace {

typedef unsigned long long u64;

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

constexpr int kCandVectors = 512;  // vectors and keys gathered before the exact bound is searched
constexpr int kCand = 1024;

struct LogprobArgs {
  const int64_t* tokens;  // nullable
  float* logprobs;        // with tokens
  float* entropy;         // nullable
  f32x4_t* stats;         // nullable: (m, log2 s, H, -) for the backward
  float* top_logprobs;    // with top > 0
  int64_t* top_ids;
  f32x4_t* part;          // segs > 1: (m, s, u, -) of each segment
  u64* keys;              // segs > 1 and top > 0: its top keys, descending, 0 where it has none
  int top, vocab;
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

// Lower bound of the `top`-th largest of the n places in LDS, by one wave:
// its first 20 bits, the rest zero. 0 where fewer than `top` are above 0.
template <int MAXN>
__device__ __forceinline__ uint32_t nth_place(const uint32_t* places, int n, int top) {
  constexpr int PER = MAXN / 64;
  uint32_t v[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int j = i * 64 + (threadIdx.x & 63);
    v[i] = j < n ? places[j] : 0u;
  }
  uint32_t bound = 0;
  for (int bit = 31; bit >= 12; --bit) {
    const uint32_t at = bound | 1u << bit;
    int c = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) c += __popcll(__ballot(v[i] >= at));
    if (c >= top) bound = at;
  }
  return bound;
}

// The keys of a segment's `top` largest logits (all where it has fewer),
// gathered in any order: a search by two bits at a time for the top-th largest
// place, then for the column up to which logits of that place belong to the
// top, the segment read again for each step. For rows of which too many logits
// reach the threshold, and for rows with NaN; element by element, so that the
// kernel's registers are those of its common rows. Reached by the whole
// workgroup; part: 64 bits a wave.
template <typename T, int TPR>
__device__ int exact_top(const T* __restrict__ row, int vocab, int seg, int span, int top, u64* cand, int* count,
                         u64* part) {
  constexpr int VE = Vec16<T>::VE;
  const RowSplit<T> sp(row, vocab);
  const int v0 = seg * span, t = threadIdx.x;
  const int end = sp.head + sp.nvec * VE;
  // the segment's columns [lo, hi), and with the first one the row's last [end, vocab)
  const int lo = seg == 0 ? 0 : sp.head + v0 * VE, hi = min(sp.head + (v0 + span) * VE, end);
  auto each = [&](auto f) {
#pragma unroll 4
    for (int i = lo + t; i < hi; i += TPR) f(place_of(to_f32(row[i])), i);
    if (seg == 0 && end + t < vocab) f(place_of(to_f32(row[end + t])), end + t);
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
#pragma unroll 4
    for (int i = 0; i < TPR / 64; ++i) c += part[i];
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

// One workgroup per segment (units by grid stride; the loop bound is uniform).
template <typename T, int VPT, int TPR, bool CAP, bool TOP>
__global__ void __launch_bounds__(TPR, VPT == 8 ? 8 : 1)
logprob_segment_kernel(const T* __restrict__ logits, int64_t rows, int64_t ld, int segs, int span, ScoreParams p,
                       LogprobArgs a) {
  constexpr int W = TPR / 64;
  __shared__ float part_m[W], part_s[W], part_u[W];
  __shared__ uint32_t places[TOP ? TPR : 1];
  __shared__ u32x4 vectors[TOP ? kCandVectors : 1];
  __shared__ int columns[TOP ? kCandVectors : 1];
  __shared__ u64 cand[TOP ? kCand : 1];
  __shared__ int count[2];  // vectors, keys
  __shared__ u64 totals[TOP ? W : 1];
  __shared__ uint32_t bound;
  for (int64_t unit = blockIdx.x; unit < rows * segs; unit += gridDim.x) {
    const int64_t row = segs == 1 ? unit : unit / segs;
    const int seg = segs == 1 ? 0 : (int)(unit - row * segs);
    const T* x = logits + row * ld;
    int64_t tok = p.ignore_index;
    float x_tok = 0.0f;
    if (segs == 1 && threadIdx.x == 0 && a.tokens) {
      tok = a.tokens[row];
      if (tok != p.ignore_index && tok >= 0 && tok < a.vocab) x_tok = to_f32(x[tok]);
    }
    Segment<T, VPT, TPR> sg(x, a.vocab, seg, span);

    const float tm = sg.largest();
    float m = wave_max(tm);
    if ((threadIdx.x & 63) == 0) part_m[threadIdx.x / 64] = m;
    int fold = 1;
    if constexpr (TOP) {
      // groups of 1, 2 or 4 threads: the fewest of at least 4 top groups
      float g = tm;
      if (TPR / 2 >= 4 * a.top) {
        g = fmaxf(g, dpp<kDppXor1>(g));
        fold = 2;
      }
      if (TPR / 4 >= 4 * a.top) {
        g = fmaxf(g, dpp<kDppXor2>(g));
        fold = 4;
      }
      // (a group that holds nothing, or -inf alone, stays below every bound)
      if (threadIdx.x % fold == 0) places[threadIdx.x / fold] = g == -INFINITY ? 0u : place_of(g);
      if (threadIdx.x < 2) count[threadIdx.x] = 0;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) m = fmaxf(m, part_m[i]);
    if constexpr (TOP) {
      if (threadIdx.x < 64) {
        const uint32_t b = fold == 4 ? nth_place<TPR / 4>(places, TPR / 4, a.top) : nth_place<TPR>(places, TPR / fold, a.top);
        if (threadIdx.x == 0) bound = b;
      }
    }
    RowStats st;
    st.m = CAP ? score<CAP>(p, m) : m;
    sg.template sums<CAP, true>(p, st.m, st.s, st.u);
    st.s = wave_sum(st.s);
    st.u = wave_sum(st.u);
    if ((threadIdx.x & 63) == 0) {
      part_s[threadIdx.x / 64] = st.s;
      part_u[threadIdx.x / 64] = st.u;
    }
    __syncthreads();
    st.s = part_s[0];
    st.u = part_u[0];
#pragma unroll
    for (int i = 1; i < W; ++i) {
      st.s += part_s[i];
      st.u += part_u[i];
    }
    if (threadIdx.x == 0) {
      if (segs == 1) finish_row<CAP>(p, a, row, st, tok, x_tok);
      else a.part[unit] = f32x4_t{st.m, st.s, st.u, 0.0f};
    }

    if constexpr (TOP) {
      constexpr int VE = Vec16<T>::VE;
      auto keep = [&](u64 key) {
        const int at = atomicAdd(&count[1], 1);
        if (at < kCand) cand[at] = key;
      };
      // vectors with a logit that reaches the threshold go to LDS whole, so
      // that their elements are looked at by as many threads
      const float least = bound == 0 ? -INFINITY : float_at(bound);
      if (tm >= least) {
        const int t = sg.thread();
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
          float vm = to_f32(sg.raw[k].e[0]);
#pragma unroll
          for (int e = 1; e < VE; ++e) vm = fmaxf(vm, to_f32(sg.raw[k].e[e]));
          if (vm >= least && t + k * TPR < sg.nv) {
            const int at = atomicAdd(&count[0], 1);
            if (at < kCandVectors) {
              vectors[at] = sg.raw[k].u;
              columns[at] = sg.col0 + (t + k * TPR) * VE;
            }
          }
        }
        if (t < sg.nx && to_f32(sg.xe) >= least) keep(key_of(to_f32(sg.xe), sg.sp.extra(t)));
      }
      __syncthreads();
      const int nvectors = count[0];
#pragma unroll 1
      for (int i = threadIdx.x; i < min(nvectors, kCandVectors) * VE; i += TPR) {
        const float v = to_f32(reinterpret_cast<const T*>(vectors)[i]);
        if (v >= least) keep(key_of(v, columns[i / VE] + i % VE));
      }
      __syncthreads();
      int n = count[1];
      if (n > kCand || nvectors > kCandVectors || st.s != st.s) {  // uniform
        n = exact_top<T, TPR>(x, a.vocab, seg, span, a.top, cand, &count[1], totals);
      }
#pragma unroll 1
      for (int c = threadIdx.x; c < n; c += TPR) {
        const u64 key = cand[c];
        int r = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) r += cand[j] > key;
        if (r < a.top) {
          if (segs == 1) store_top<CAP>(p, a, row, r, key, st);
          else a.keys[unit * a.top + r] = key;
        }
      }
      if (segs > 1)
        for (int r = n + threadIdx.x; r < a.top; r += TPR) a.keys[unit * a.top + r] = 0;
    }
    __syncthreads();  // the shared arrays are rewritten for the workgroup's next unit
  }
}

// Joins a row's segments: wave 0 folds the statistics in a fixed order; with
// alternatives, the top-th largest key among the segments' j-th keys, j the
// fewest that make top of them, bounds the row's top from below, and what
// reaches it is placed by counting.
constexpr int kJoinThreads = 256;

template <typename T, bool CAP>
__global__ void __launch_bounds__(kJoinThreads)
logprob_join_kernel(const T* __restrict__ logits, int64_t ld, int segs, ScoreParams p, LogprobArgs a) {
  __shared__ RowStats whole;
  __shared__ u64 cand[kJoinKeys];
  __shared__ int count;
  __shared__ u64 low;
  const int64_t row = blockIdx.x;
  const int t = threadIdx.x;
  if (t == 0) {
    count = 0;
    low = 0;
  }
  if (t < 64) {
    int64_t tok = p.ignore_index;
    float x_tok = 0.0f;
    if (t == 0 && a.tokens) {
      tok = a.tokens[row];
      if (tok != p.ignore_index && tok >= 0 && tok < a.vocab) x_tok = to_f32(logits[row * ld + tok]);
    }
    RowStats st{-INFINITY, 0.0f, 0.0f};
    for (int i = t; i < segs; i += 64) {
      const f32x4_t q = a.part[row * segs + i];
      st = join_stats(p, st, RowStats{q[0], q[1], q[2]});
    }
    st = wave_join(p, st);
    if (t == 0) {
      whole = st;
      finish_row<CAP>(p, a, row, st, tok, x_tok);
    }
  }
  if (a.top == 0) return;
  __syncthreads();
  const RowStats st = whole;
  const u64* keys = a.keys + row * segs * a.top;
  const int j = (a.top - 1) / segs;
  for (int i = t; i < segs; i += kJoinThreads) cand[i] = keys[i * a.top + j];
  __syncthreads();
  // the rank of the bound among the segs keys: the (j + 1) segs' worth of keys above or at it number top at least
  const int rank = (a.top - 1) / (j + 1);
  for (int i = t; i < segs; i += kJoinThreads) {
    const u64 key = cand[i];
    int r = 0;
    for (int k = 0; k < segs; ++k) r += cand[k] > key || (cand[k] == key && k < i);
    if (r == rank) low = key;
  }
  __syncthreads();
  const u64 least = low;
  for (int i = t; i < segs * a.top; i += kJoinThreads) {
    const u64 key = keys[i];
    if (key >= least && key != 0) cand[atomicAdd(&count, 1)] = key;
  }
  __syncthreads();
  const int n = count;
#pragma unroll 1
  for (int c = t; c < n; c += kJoinThreads) {
    const u64 key = cand[c];
    int r = 0;
#pragma unroll 4
    for (int k = 0; k < n; ++k) r += cand[k] > key;
    if (r < a.top) store_top<CAP>(p, a, row, r, key, st);
  }
}

// The gradient from the forward's statistics; blockIdx.y takes `span` vectors
// of the row. The given token's entry is written again, with its own term,
// once the row's others have left.
template <typename T, bool CAP, bool NT, int U>
__global__ void __launch_bounds__(kGradThreads)
logprob_grad_kernel(const T* __restrict__ logits, const int64_t* __restrict__ tokens, const f32x4_t* __restrict__ stats,
                    const float* __restrict__ g_logprobs, const float* __restrict__ g_entropy, T* __restrict__ grad,
                    int64_t rows, int vocab, int64_t ld, int64_t ld_g, int span, ScoreParams p) {
  const int v0 = blockIdx.y * span, v1 = v0 + span;
  const bool ends = blockIdx.y == 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* x = logits + row * ld;
    T* gx = grad + row * ld_g;
    const f32x4_t st = stats[row];
    const int64_t tok = tokens ? tokens[row] : -1;
    const bool ignored = tokens && tok == p.ignore_index;
    const bool bad = tokens && !ignored && (tok < 0 || tok >= vocab);
    const bool empty = st[0] == -INFINITY && st[1] == 0.0f;
    if (ignored || empty) {  // whatever the row holds
      map_row<T, NT, 1>(x, gx, vocab, v0, v1, ends, [](float) { return 0.0f; });
      continue;
    }
    const float g = bad ? NAN : (tokens && g_logprobs ? g_logprobs[row] : 0.0f);
    const float e = g_entropy ? g_entropy[row] : 0.0f;
    const float m = st[0], l2 = st[1];
    // -(g + e (ln p + H)) = c0 + c1 log2 p
    const float c0 = -fmaf(e, st[2], g), c1 = -e * kLn2;
    auto dense = [&](float v) {
      float slope;
      const float y = score_and_slope<CAP>(p, v, slope);
      const float lp = (y - m) * p.c2 - l2;
      // p is 0 from -150 on, and log2 p may be -inf there
      return __builtin_amdgcn_exp2f(lp) * fmaf(c1, fmaxf(lp, -1000.0f), c0) * slope;
    };
    map_row<T, NT, U>(x, gx, vocab, v0, v1, ends, dense);
    if (tokens && !bad && wrote_column(x, vocab, v0, v1, ends, (int)tok)) {  // uniform
      stores_done();
      if (threadIdx.x == 0) {
        float slope;
        const float v = to_f32(x[tok]);
        score_and_slope<CAP>(p, v, slope);
        gx[tok] = from_f32<T>(fmaf(g, slope, dense(v)));
      }
    }
  }
}

struct Workspace {
  size_t part, keys, total;
};

Workspace workspace(int64_t rows, const ScorePlan& pl, int top) {
  auto up = [](size_t v) { return (v + 255) & ~(size_t)255; };
  Workspace w{0, 0, 0};
  if (pl.segs == 1 || rows <= 0) return w;
  w.keys = up((size_t)rows * pl.segs * sizeof(f32x4_t));
  w.total = w.keys + up((size_t)rows * pl.segs * top * sizeof(u64));
  return w;
}

template <typename T, bool CAP>
void launch_fwd(const void* logits, int64_t rows, int64_t ld, const ScorePlan& pl, const ScoreParams& p,
                const LogprobArgs& a, hipStream_t s) {
  const T* x = static_cast<const T*>(logits);
  const dim3 grid(row_grid(rows * pl.segs));
#define GO(VPT, TPR)                                                                                           \
  (a.top ? logprob_segment_kernel<T, VPT, TPR, CAP, true><<<grid, dim3(TPR), 0, s>>>(x, rows, ld, pl.segs, pl.span, p, a) \
         : logprob_segment_kernel<T, VPT, TPR, CAP, false><<<grid, dim3(TPR), 0, s>>>(x, rows, ld, pl.segs, pl.span, p, a))
  AK_SEGMENT_DISPATCH(pl.span, GO);
#undef GO
  if (pl.segs > 1) logprob_join_kernel<T, CAP><<<dim3((unsigned)rows), dim3(a.top ? kJoinThreads : 64), 0, s>>>(x, ld, pl.segs, p, a);
}

template <typename T, bool CAP>
void launch_bwd(const void* logits, const int64_t* tokens, const float* stats, const float* gl, const float* ge,
                void* grad, int64_t rows, int vocab, int64_t ld, int64_t ld_g, const ScoreParams& p, hipStream_t s) {
  constexpr int VE = Vec16<T>::VE;
  const ScorePlan pl = grad_plan(vocab, VE);
  const dim3 grid(row_grid(rows), pl.segs), block(kGradThreads);
  const T* x = static_cast<const T*>(logits);
  T* g = static_cast<T*>(grad);
  const f32x4_t* st = reinterpret_cast<const f32x4_t*>(stats);
  if (vocab / VE < 4 * kGradThreads)
    logprob_grad_kernel<T, CAP, false, 1><<<grid, block, 0, s>>>(x, tokens, st, gl, ge, g, rows, vocab, ld, ld_g, pl.span, p);
  else if (score_past_cache(2 * rows * vocab * (int64_t)sizeof(T)))
    logprob_grad_kernel<T, CAP, true, 4><<<grid, block, 0, s>>>(x, tokens, st, gl, ge, g, rows, vocab, ld, ld_g, pl.span, p);
  else
    logprob_grad_kernel<T, CAP, false, 4><<<grid, block, 0, s>>>(x, tokens, st, gl, ge, g, rows, vocab, ld, ld_g, pl.span, p);
}

}  // namespace
}  // namespace ak

extern "C" size_t ak_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int top_k, int dtype) {
  const int esz = ak_dtype_size(dtype);
  if (rows <= 0 || vocab <= 0 || vocab > ak::kScoreVocab || top_k < 0 || top_k > ak::kMaxTop || esz == 0) return 0;
  return ak::workspace(rows, ak::score_plan(rows, vocab, 16 / esz, top_k), top_k).total;
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
  const ak::ScorePlan pl = ak::score_plan(rows, vocab, 16 / ak_dtype_size(dtype), top_k);
  const ak::Workspace w = ak::workspace(rows, pl, top_k);
  if (workspace_bytes < w.total || (w.total && (!workspace || !ak::aligned16(workspace))))
    return ak_set_error(AK_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed (16-byte aligned)", name, workspace_bytes, w.total);
  char* ws = static_cast<char*>(workspace);
  const ak::LogprobArgs a{tokens, logprobs, entropy, reinterpret_cast<ak::f32x4_t*>(stats), top_logprobs, top_ids,
                          reinterpret_cast<ak::f32x4_t*>(ws), reinterpret_cast<ak::u64*>(ws + w.keys), top_k, (int)vocab};
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
