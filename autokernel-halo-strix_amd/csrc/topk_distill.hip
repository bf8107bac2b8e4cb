// Distillation from a teacher's top logits, for gfx950.
//
//   y = softcap > 0 ? softcap * tanh(x / softcap) : x,  p = softmax(y / T) over the vocabulary
//   q = softmax(teacher / T) over the row's given entries (at most 256)
//   loss  = T^2 sum_k q_k (ln q_k - ln p[id_k])
//   dx_v  = g T^2 (p_v - sum of q_k with id_k == v) (1 - tanh^2) / T
// An entry whose id is ignore_index is not there; a row without entries has
// loss 0, a zero gradient and no part in the mean. The same id twice counts
// twice.
//
// HBM-bound: the forward reads the student's logits once (score_rows.h), one
// wave a row adds the teacher's entries; the backward reads the logits once
// more and writes the gradient once. Writing the gradient in the forward would
// save that read where the upstream gradient is exactly 1, but such a loss is
// weighted against another (or scaled, in fp16): the stored gradient would
// then be read, scaled, rounded a second time and written again. Measured (a copy
// of 1 GiB here: 5.1 TB/s): [4096, 32768] bf16 with 64 entries 51 us forward and
// 85 us backward, 5.2 and 6.3 TB/s; [1999, 50257] fp32 with 128 entries and a
// softcap 90 and 130 us.
#include "score_rows.h"

namespace ak {
namespace {

constexpr int kPerLane = kMaxTop / 64;  // a row's entries held by one wave

struct TeacherArgs {
  const void* logits;  // [rows, top] of dtype `code`
  const int64_t* ids;  // [rows, top]
  int64_t ld, ld_ids;
  int top, code, vocab;
  float t2;            // temperature^2
};

__device__ __forceinline__ float teacher_logit(const TeacherArgs& a, int64_t row, int k) {
  const int64_t at = row * a.ld + k;
  if (a.code == AK_DTYPE_F32) return static_cast<const float*>(a.logits)[at];
  if (a.code == AK_DTYPE_F16) return to_f32(static_cast<const f16*>(a.logits)[at]);
  return to_f32(static_cast<const bf16*>(a.logits)[at]);
}

// One row's entries in one wave. The loads are issued where it is made, and
// used in `entries` and `student`, so that a row's own loads may come between.
struct RawEntries {
  float t[kPerLane];
  int64_t id[kPerLane];
  __device__ __forceinline__ RawEntries(const TeacherArgs& a, int64_t row, int top) {
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const int k = (threadIdx.x & 63) + 64 * i;
      if (64 * i >= top) continue;  // uniform
      id[i] = a.ids[row * a.ld_ids + min(k, top - 1)];
      t[i] = teacher_logit(a, row, min(k, top - 1));
    }
  }
};

// -inf where there is no entry.
template <typename T>
struct Entries {
  float t[kPerLane], x[kPerLane];  // the teacher's logits, the student's
  bool bad;                        // an id outside the vocabulary
  __device__ __forceinline__ Entries(const TeacherArgs& a, const RawEntries& r, const T* __restrict__ row, int64_t ignore_index,
                                     int top) {
    bad = false;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      t[i] = -INFINITY;
      x[i] = 0.0f;
      if (64 * i >= top) continue;  // uniform
      const bool here = (int)(threadIdx.x & 63) + 64 * i < top && r.id[i] != ignore_index;
      const bool in = r.id[i] >= 0 && r.id[i] < a.vocab;
      bad |= here && !in;
      t[i] = here && in ? r.t[i] : -INFINITY;
      x[i] = to_f32(row[here && in ? r.id[i] : 0]);
    }
  }
};

// Loss of a row, by one wave. out: (m, log2 s, the largest teacher logit, log2
// of the sum of 2^((t - largest) c2)) for the backward; m is NaN where the
// loss is.
template <typename T, bool CAP>
__device__ __forceinline__ void finish_row(const ScoreParams& p, const TeacherArgs& a, int64_t row, const RowStats& st,
                                           const Entries<T>& en, float* __restrict__ losses,
                                           f32x4_t* __restrict__ out) {
  float tm = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) tm = fmaxf(tm, en.t[i]);
  tm = wave_max(tm);
  const bool any_bad = __any(en.bad);
  bool nan = false;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) nan |= en.t[i] != en.t[i];
  nan = __any(nan) || any_bad;
  float loss = 0.0f, tl = 0.0f, m = st.m;
  const float l2 = log2_sum(st);
  if (nan) {
    loss = m = NAN;
    tm = 0.0f;
  } else if (tm != -INFINITY) {
    float ts = 0.0f;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) ts += __builtin_amdgcn_exp2f((en.t[i] - tm) * p.c2);
    tl = __builtin_amdgcn_logf(wave_sum(ts));
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const float lq = (en.t[i] - tm) * p.c2 - tl;
      const float q = __builtin_amdgcn_exp2f(lq);
      if (q != 0.0f) loss += q * (kLn2 * lq - log_prob(p, score<CAP>(p, en.x[i]), st.m, l2));
    }
    loss = wave_sum(loss) * a.t2;
    if (loss != loss) m = NAN;
  }
  if ((threadIdx.x & 63) == 0) {
    losses[row] = loss;
    out[row] = f32x4_t{m, l2, tm, tl};
  }
}

// One workgroup per segment (units by grid stride; the loop bound is uniform).
template <typename T, int VPT, int TPR, bool CAP>
__global__ void __launch_bounds__(TPR, AK_SEGMENT_WAVES(VPT))
distill_segment_kernel(const T* __restrict__ logits, int64_t rows, int64_t ld, int segs, int span, ScoreParams p,
                       TeacherArgs a, float* __restrict__ losses, f32x4_t* __restrict__ stats,
                       f32x4_t* __restrict__ part) {
  constexpr int W = TPR / 64;
  __shared__ float part_m[W], part_s[W];
  for (int64_t unit = blockIdx.x; unit < rows * segs; unit += gridDim.x) {
    const int64_t row = segs == 1 ? unit : unit / segs;
    const int seg = segs == 1 ? 0 : (int)(unit - row * segs);
    const T* x = logits + row * ld;
    // (the other waves' loads of the entries hit the same lines)
    const int entries = segs == 1 ? a.top : 0;
    const RawEntries raw(a, row, entries);
    Segment<T, VPT, TPR> sg(x, a.vocab, seg, span);
    const Entries<T> en(a, raw, x, p.ignore_index, entries);
    float m = wave_max(sg.largest());
    if ((threadIdx.x & 63) == 0) part_m[threadIdx.x / 64] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) m = fmaxf(m, part_m[i]);
    RowStats st;
    st.m = CAP ? score<CAP>(p, m) : m;
    sg.template sums<CAP, false>(p, st.m, st.s, st.u);
    st.s = wave_sum(st.s);
    if ((threadIdx.x & 63) == 0) part_s[threadIdx.x / 64] = st.s;
    __syncthreads();  // part_m has been read by all, so the next unit may write it
    st.s = part_s[0];
#pragma unroll
    for (int i = 1; i < W; ++i) st.s += part_s[i];
    if (segs > 1) {
      if (threadIdx.x == 0) part[unit] = f32x4_t{st.m, st.s, 0.0f, 0.0f};
    } else if (threadIdx.x < 64) {
      finish_row<T, CAP>(p, a, row, st, en, losses, stats);
    }
    __syncthreads();  // part_s is rewritten for the workgroup's next unit
  }
}

// Joins a row's segments, one wave a row.
template <typename T, bool CAP>
__global__ void __launch_bounds__(64)
distill_join_kernel(const T* __restrict__ logits, int64_t row0, int64_t ld, int segs, ScoreParams p, TeacherArgs a,
                    float* __restrict__ losses, f32x4_t* __restrict__ stats, const f32x4_t* __restrict__ part) {
  const int64_t row = row0 + blockIdx.x;
  const Entries<T> en(a, RawEntries(a, row, a.top), logits + row * ld, p.ignore_index, a.top);
  RowStats st{-INFINITY, 0.0f, 0.0f};
  for (int i = threadIdx.x; i < segs; i += 64) {
    const f32x4_t q = part[row * segs + i];
    st = join_stats(p, st, RowStats{q[0], q[1], 0.0f});
  }
  st = wave_join(p, st);
  finish_row<T, CAP>(p, a, row, st, en, losses, stats);
}

// loss[0] = sum of losses / max(1, #rows with entries), scale[0] = 1 / that
// divisor; one workgroup, in a fixed order.
constexpr int kMeanThreads = 1024;

__global__ void __launch_bounds__(kMeanThreads)
distill_mean_kernel(const float* __restrict__ losses, const f32x4_t* __restrict__ stats, int64_t rows,
                    float* __restrict__ loss, float* __restrict__ scale) {
  __shared__ float part_s[kMeanThreads / 64], part_n[kMeanThreads / 64];
  float s = 0.0f;
  int n = 0;
  for (int64_t i = threadIdx.x; i < rows; i += kMeanThreads) {
    s += losses[i];
    n += stats[i][2] != -INFINITY;
  }
  s = wave_sum(s);
  for (int off = 32; off >= 1; off >>= 1) n += __shfl_xor(n, off, 64);
  if ((threadIdx.x & 63) == 0) {
    part_s[threadIdx.x / 64] = s;
    part_n[threadIdx.x / 64] = (float)n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    float c = part_n[0];
    s = part_s[0];
    for (int i = 1; i < kMeanThreads / 64; ++i) {
      s += part_s[i];
      c += part_n[i];
    }
    c = fmaxf(c, 1.0f);
    loss[0] = s / c;
    scale[0] = 1.0f / c;
  }
}

constexpr int kSlots = kSpan + 16;  // a span's vectors, and the elements around the vectors

// (p_v - q_v) c. In LDS: for each vector of the span, and each single element,
// 1 + the first of its entries, or 0; each entry's column, gradient and the
// vector's next entry.
template <typename T, bool CAP>
struct DistillRow {
  const ScoreParams& p;
  float m, l2, c;
  const uint32_t* first;
  const int* ids;
  const float* grads;
  const uint32_t* next;
  __device__ __forceinline__ float value(float x, float q) const {
    float slope;
    const float y = score_and_slope<T, CAP>(p, x, slope);
    return (__builtin_amdgcn_exp2f((y - m) * p.c2 - l2) - q) * (c * slope);
  }
  __device__ __forceinline__ float many(float x) const { return value(x, 0.0f); }
  __device__ __forceinline__ float one(float x, int, int i) const {
    const uint32_t k = first[kSpan + i];
    return k ? grads[k - 1] : value(x, 0.0f);
  }
  __device__ __forceinline__ void patch(const Vec16<T>&, int col, int v, Vec16<T>& o) const {
    for (uint32_t k = first[v]; k; k = next[k - 1]) {
      const int at = ids[k - 1] - col;
      const T g = from_f32<T>(grads[k - 1]);
#pragma unroll
      for (int e = 0; e < Vec16<T>::VE; ++e) o.e[e] = e == at ? g : o.e[e];
    }
  }
};

// The gradient from the forward's statistics; a workgroup takes `span` vectors of
// a row. The entries of the span are worked out first, a thread each, and put
// into their vectors' results on the way out. (Written over the stored row
// instead, they cost [4096, 50257] bf16 with 64 entries 50 us behind a barrier
// that waits for all stores, 30 us in a launch of their own, and 40 us where
// each vector's thread works its entries out.)
template <typename T, bool CAP, bool NT, int U>
__global__ void __launch_bounds__(kGradThreads)
distill_grad_kernel(const T* __restrict__ logits, const f32x4_t* __restrict__ stats, const float* __restrict__ g_loss,
                    int64_t g_stride, const float* __restrict__ scale, T* __restrict__ grad, int64_t rows,
                    int64_t ld, int64_t ld_g, int spans, int span, ScoreParams p, TeacherArgs a) {
  constexpr int VE = Vec16<T>::VE;
  __shared__ uint32_t first[kSlots], next[kMaxTop];
  __shared__ int ids[kMaxTop];
  __shared__ float qs[kMaxTop], grads[kMaxTop];
  const int t = threadIdx.x;
  static_assert(kMaxTop <= kGradThreads, "an entry a thread");
  for (int64_t unit = blockIdx.x; unit < rows * spans; unit += gridDim.x) {
    const int64_t row = unit / spans;
    const int v0 = (int)(unit - row * spans) * span, v1 = v0 + span;
    const bool ends = v0 == 0;
    const T* x = logits + row * ld;
    T* gx = grad + row * ld_g;
    const f32x4_t st = stats[row];
    if (st[2] == -INFINITY) {  // no entries
      map_row<T, NT, 1>(x, gx, a.vocab, v0, v1, ends, ZeroRow());
      continue;
    }
    const RowSplit<T> sp(x, a.vocab);
    int slot = -1;  // of this thread's entry, if this workgroup writes its column
    float xv = 0.0f;
    if (t < a.top) {
      const int64_t id = a.ids[row * a.ld_ids + t];
      const bool there = id != p.ignore_index && id >= 0 && id < a.vocab;
      qs[t] = __builtin_amdgcn_exp2f((teacher_logit(a, row, t) - st[2]) * p.c2 - st[3]);
      ids[t] = there ? (int)id : -1;
      if (there) {
        const int c = (int)id - sp.head, v = c / VE;
        if (c < 0 || v >= sp.nvec) slot = ends ? kSpan + (c < 0 ? (int)id : (int)id - sp.nvec * VE) : -1;
        else if (v >= v0 && v < v1) slot = v - v0;
        if (slot >= 0) xv = to_f32(x[id]);
      }
    }
    for (int i = t; i < span; i += kGradThreads) first[i] = 0;
    if (t < 16) first[kSpan + t] = 0;
    __syncthreads();
    const DistillRow<T, CAP> f{p, st[0] == -INFINITY ? 0.0f : st[0], st[1],
                               g_loss[row * g_stride] * (scale ? scale[0] : 1.0f) * a.t2, first, ids, grads, next};
    if (slot >= 0) next[t] = atomicExch(&first[slot], (uint32_t)t + 1);
    __syncthreads();
    if (slot >= 0) {
      // equal ids are in one list: their sum, in the order of the entries, whatever the list's
      float q = 0.0f;
      for (uint32_t last = 0, least; last <= kMaxTop; last = least) {
        least = kMaxTop + 1;
        for (uint32_t k = first[slot]; k; k = next[k - 1])
          if (k > last && ids[k - 1] == ids[t]) least = min(least, k);
        if (least <= kMaxTop) q += qs[least - 1];
      }
      grads[t] = f.value(xv, q);
    }
    __syncthreads();
    map_row<T, NT, U>(x, gx, a.vocab, v0, v1, ends, f);
    __syncthreads();  // the arrays are rewritten for the workgroup's next row
  }
}

size_t part_bytes(int64_t rows, const ScorePlan& pl) {
  return pl.segs > 1 && rows > 0 ? ((size_t)rows * pl.segs * sizeof(f32x4_t) + 255) & ~(size_t)255 : 0;
}

template <typename T, bool CAP>
void launch_fwd(const void* logits, int64_t rows, int64_t ld, const ScorePlan& pl, const ScoreParams& p,
                const TeacherArgs& a, float* losses, float* stats, void* ws, hipStream_t s) {
  const T* x = static_cast<const T*>(logits);
  f32x4_t* st = reinterpret_cast<f32x4_t*>(stats);
  f32x4_t* part = static_cast<f32x4_t*>(ws);
  const dim3 grid(row_grid(rows * pl.segs));
#define GO(VPT, TPR) \
  distill_segment_kernel<T, VPT, TPR, CAP><<<grid, dim3(TPR), 0, s>>>(x, rows, ld, pl.segs, pl.span, p, a, losses, st, part)
  AK_SEGMENT_DISPATCH(pl.span, GO);
#undef GO
  for (int64_t row0 = 0; pl.segs > 1 && row0 < rows; row0 += kMaxRowGrid)
    distill_join_kernel<T, CAP><<<dim3(row_grid(rows - row0)), dim3(64), 0, s>>>(x, row0, ld, pl.segs, p, a, losses, st, part);
}

template <typename T, bool CAP>
void launch_bwd(const void* logits, const float* stats, const float* g_loss, int64_t g_stride, const float* scale,
                void* grad, int64_t rows, int64_t ld, int64_t ld_g, const ScoreParams& p, const TeacherArgs& a,
                hipStream_t s) {
  constexpr int VE = Vec16<T>::VE;
  const ScorePlan pl = grad_plan(a.vocab, VE);
  const dim3 grid(row_grid(rows * pl.segs)), block(kGradThreads);
  const T* x = static_cast<const T*>(logits);
  T* g = static_cast<T*>(grad);
  const f32x4_t* st = reinterpret_cast<const f32x4_t*>(stats);
  if (a.vocab / VE < 4 * kGradThreads)
    distill_grad_kernel<T, CAP, false, 1><<<grid, block, 0, s>>>(x, st, g_loss, g_stride, scale, g, rows, ld, ld_g, pl.segs, pl.span, p, a);
  else if (score_past_cache(2 * rows * a.vocab * (int64_t)sizeof(T)))
    distill_grad_kernel<T, CAP, true, 4><<<grid, block, 0, s>>>(x, st, g_loss, g_stride, scale, g, rows, ld, ld_g, pl.segs, pl.span, p, a);
  else
    distill_grad_kernel<T, CAP, false, 4><<<grid, block, 0, s>>>(x, st, g_loss, g_stride, scale, g, rows, ld, ld_g, pl.segs, pl.span, p, a);
}

int check(const char* name, const void* logits, const void* teacher, const int64_t* ids, int64_t rows, int64_t vocab,
          int64_t top, int64_t ld, int64_t ld_t, int64_t ld_ids, float temperature, float softcap, int dtype,
          int teacher_dtype) {
  const int rc = check_score_rows(name, rows, vocab, ld, temperature, softcap, dtype);
  if (rc) return rc;
  if (ak_dtype_size(teacher_dtype) == 0) return ak_set_error(AK_ERR_UNSUPPORTED, "%s: unsupported teacher dtype code %d", name, teacher_dtype);
  if (top < 1 || top > kMaxTop)
    return ak_set_error(AK_ERR_INVALID_ARG, "%s: %lld teacher entries a row, 1 to %d are taken", name, (long long)top, kMaxTop);
  if (ld_t < top || ld_ids < top) return ak_set_error(AK_ERR_INVALID_ARG, "%s: row pitch smaller than the entries", name);
  if (!ak_extent_ok(rows, ld_t, top, 4) || !ak_extent_ok(rows, ld_ids, top, 8))
    return ak_set_error(AK_ERR_INVALID_ARG, "%s: rows=%lld x pitch exceed 64-bit addressing", name, (long long)rows);
  if (rows > 0 && (!logits || !teacher || !ids)) return ak_set_error(AK_ERR_INVALID_ARG, "%s: null pointer", name);
  return AK_OK;
}

}  // namespace
}  // namespace ak

extern "C" size_t ak_topk_distill_workspace_bytes(int64_t rows, int64_t vocab, int dtype) {
  const int esz = ak_dtype_size(dtype);
  if (rows <= 0 || vocab <= 0 || vocab > ak::kScoreVocab || esz == 0) return 0;
  return ak::part_bytes(rows, ak::score_plan(rows, vocab, 16 / esz));
}

extern "C" int ak_topk_distill_fwd(const void* logits, const void* teacher_logits, const int64_t* teacher_ids,
                                   float* losses, float* stats, float* loss, float* scale, void* workspace,
                                   size_t workspace_bytes, int64_t rows, int64_t vocab, int64_t top, int64_t ld_logits,
                                   int64_t ld_teacher, int64_t ld_ids, float temperature, float softcap,
                                   int64_t ignore_index, int dtype, int teacher_dtype, void* stream) {
  const char* name = "ak_topk_distill_fwd";
  const int rc = ak::check(name, logits, teacher_logits, teacher_ids, rows, vocab, top, ld_logits, ld_teacher, ld_ids,
                           temperature, softcap, dtype, teacher_dtype);
  if (rc) return rc;
  if (!loss != !scale || (rows > 0 && (!losses || !stats))) return ak_set_error(AK_ERR_INVALID_ARG, "%s: null pointer", name);
  if (stats && !ak::aligned16(stats)) return ak_set_error(AK_ERR_INVALID_ARG, "%s: stats must be 16-byte aligned", name);
  if (rows == 0 && !loss) return AK_OK;
  hipStream_t s = ak_stream(stream);
  if (rows > 0) {
    const ak::ScorePlan pl = ak::score_plan(rows, vocab, 16 / ak_dtype_size(dtype));
    const size_t need = ak::part_bytes(rows, pl);
    if (workspace_bytes < need || (need && (!workspace || !ak::aligned16(workspace))))
      return ak_set_error(AK_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed (16-byte aligned)", name, workspace_bytes, need);
    const ak::ScoreParams p = ak::score_params(temperature, softcap, ignore_index);
    const ak::TeacherArgs a{teacher_logits, teacher_ids, ld_teacher, ld_ids, (int)top, teacher_dtype, (int)vocab,
                            temperature * temperature};
    auto go = [&](auto t) {
      using T = decltype(t);
      if (softcap > 0.0f) ak::launch_fwd<T, true>(logits, rows, ld_logits, pl, p, a, losses, stats, workspace, s);
      else ak::launch_fwd<T, false>(logits, rows, ld_logits, pl, p, a, losses, stats, workspace, s);
    };
    if (dtype == AK_DTYPE_F32) go(float());
    else if (dtype == AK_DTYPE_F16) go(ak::f16());
    else go(ak::bf16());
  }
  if (loss)
    ak::distill_mean_kernel<<<dim3(1), dim3(ak::kMeanThreads), 0, s>>>(losses, reinterpret_cast<ak::f32x4_t*>(stats), rows, loss, scale);
  return ak_check_launch(name);
}

extern "C" int ak_topk_distill_bwd(const void* logits, const void* teacher_logits, const int64_t* teacher_ids,
                                   const float* stats, const float* grad_loss, int64_t grad_stride, const float* scale,
                                   void* grad_logits, int64_t rows, int64_t vocab, int64_t top, int64_t ld_logits,
                                   int64_t ld_teacher, int64_t ld_ids, int64_t ld_grad, float temperature,
                                   float softcap, int64_t ignore_index, int dtype, int teacher_dtype, void* stream) {
  const char* name = "ak_topk_distill_bwd";
  int rc = ak::check(name, logits, teacher_logits, teacher_ids, rows, vocab, top, ld_logits, ld_teacher, ld_ids,
                     temperature, softcap, dtype, teacher_dtype);
  if (!rc) rc = ak::check_score_rows(name, rows, vocab, ld_grad, temperature, softcap, dtype);
  if (rc) return rc;
  if (grad_stride != 0 && grad_stride != 1) return ak_set_error(AK_ERR_INVALID_ARG, "%s: grad_stride must be 0 or 1", name);
  if (rows == 0) return AK_OK;
  if (!stats || !grad_loss || !grad_logits) return ak_set_error(AK_ERR_INVALID_ARG, "%s: null pointer", name);
  if (!ak::aligned16(stats)) return ak_set_error(AK_ERR_INVALID_ARG, "%s: stats must be 16-byte aligned", name);
  const ak::ScoreParams p = ak::score_params(temperature, softcap, ignore_index);
  const ak::TeacherArgs a{teacher_logits, teacher_ids, ld_teacher, ld_ids, (int)top, teacher_dtype, (int)vocab,
                          temperature * temperature};
  hipStream_t s = ak_stream(stream);
  auto go = [&](auto t) {
    using T = decltype(t);
    if (softcap > 0.0f) ak::launch_bwd<T, true>(logits, stats, grad_loss, grad_stride, scale, grad_logits, rows, ld_logits, ld_grad, p, a, s);
    else ak::launch_bwd<T, false>(logits, stats, grad_loss, grad_stride, scale, grad_logits, rows, ld_logits, ld_grad, p, a, s);
  };
  if (dtype == AK_DTYPE_F32) go(float());
  else if (dtype == AK_DTYPE_F16) go(ak::f16());
  else go(ak::bf16());
  return ak_check_launch(name);
}
