// Attention of new tokens over a paged cache, for gfx950.
//
//   s_j = scale q . k_j          (softcap > 0: softcap tanh(s_j / softcap))
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   m = max_j s_j
// over the keys j that the token at position p sees: j <= p, j > p - window where
// there is a window, j below the sequence's length, on a page that exists. One
// pass over the keys with the running maximum and sum; where the keys of a row
// are cut among workers, each leaves (m, sum, sum of products) in fp32 and a
// second kernel joins them in a fixed order. A row that sees nothing, or only
// scores of -inf, is 0.
#include <algorithm>

#include "paged_attention.h"

namespace ak {
namespace {

// What the tiles do not take, heads of more than 256 elements, rows that are not
// of whole aligned vectors, very many query heads to a key head: a workgroup for
// a row (token and query head) and a cut of its keys. A wave takes 64 keys at a
// time: a lane each for the scores, then a lane for every 64th element of the
// values' sum. Bound by the strided reads of the keys: 16 sequences of
// 1024 to 4096 keys, 32 + 8 heads of 128 bf16, off the alignment, 1270 us, in tiles 49 to 54.
template <typename T>
__global__ void __launch_bounds__(256) attend_any_kernel(AttendArgs a, int64_t rows) {
  constexpr int kPer = kMaxAttendDim / 64;
  __shared__ float qf[kMaxAttendDim];
  __shared__ float prob[4][64];
  __shared__ float sums[4][kMaxAttendDim];
  __shared__ float stat[4][2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float factor = score_factor(a);
  // (a row's sums are read before the next row's first barrier, and written after it)
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const int64_t token = (uint32_t)row / (uint32_t)a.q_heads;
    const int h = (int)(row - token * a.q_heads), kvh = h / (a.q_heads / a.kv_heads);
    const int b = sequence_of(a.seq, (int)token);
    int64_t lo = 0, hi = 0;
    if (b >= 0) {
      int first, count;
      sequence_tokens(a.seq, b, first, count);
      const int64_t length = a.seq.lengths[b];
      keys_of(a, length, length - count + (token - first), lo, hi);
    }
    // this workgroup's cut, in whole blocks of 64
    const int64_t blocks = (hi - lo + 63) / 64;
    const int64_t end = min(hi, lo + blocks * (blockIdx.y + 1) / a.splits * 64);
    lo += blocks * blockIdx.y / a.splits * 64;
    hi = end;
    const T* q = static_cast<const T*>(a.q) + token * a.q_st + h * a.q_sh;
    for (int d = threadIdx.x; d < a.dim; d += 256) qf[d] = to_f32(q[d]);
    __syncthreads();
    float m = kNegInf, l = 0.0f, acc[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] = 0.0f;
    for (int64_t j0 = lo + wave * 64; j0 < hi; j0 += 256) {
      const int64_t j = j0 + lane;
      int64_t slot = 0, page = -1;
      if (j < hi) page = page_of(a, b, j, slot);
      float s = kNegInf;
      if (page >= 0) {
        const T* k = static_cast<const T*>(a.k) + page * a.kp + slot * a.ks + kvh * a.kh;
        float dot = 0.0f;
        for (int d = 0; d < a.dim; ++d) dot = fmaf(qf[d], to_f32(k[d]), dot);
        s = score_of(a, dot);
      }
      const float top = fmaxf(m, wave_max(s));
      const float p = page >= 0 ? weight_of(s, top, factor) : 0.0f;
      const float keep = weight_of(m, top, factor);
      m = top;
      l = l * keep + p;
      prob[wave][lane] = p;
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int i = 0; i < kPer; ++i) acc[i] *= keep;
      uint64_t seen = __ballot(page >= 0);  // masked values take no part, whatever they hold
      while (seen) {
        const int x = __builtin_ctzll(seen);
        seen &= seen - 1;
        const int64_t vpage = __shfl(page, x), vslot = __shfl(slot, x);
        const T* v = static_cast<const T*>(a.v) + vpage * a.vp + vslot * a.vs + kvh * a.vh;
        const float px = prob[wave][x];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          if (i * 64 < a.dim && i * 64 + lane < a.dim) acc[i] = fmaf(px, to_f32(v[i * 64 + lane]), acc[i]);
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
    l = wave_sum(l);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (i * 64 + lane < a.dim) sums[wave][i * 64 + lane] = acc[i];
    if (lane == 0) {
      stat[wave][0] = m;
      stat[wave][1] = l;
    }
    __syncthreads();
    float top = kNegInf, total = 0.0f, f[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, stat[w][0]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      f[w] = weight_of(stat[w][0], top, factor);
      total += f[w] * stat[w][1];
    }
    if (a.splits > 1) {
      float* part = a.part + (row * a.splits + blockIdx.y) * (a.dim + 2);
      for (int d = threadIdx.x; d < a.dim; d += 256)
        part[d] = f[0] * sums[0][d] + f[1] * sums[1][d] + f[2] * sums[2][d] + f[3] * sums[3][d];
      if (threadIdx.x == 0) {
        part[a.dim] = top;
        part[a.dim + 1] = total;
      }
      continue;
    }
    if (b < 0 && !a.zero_other) continue;
    T* out = static_cast<T*>(a.out) + token * a.o_st + h * a.o_sh;
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    for (int d = threadIdx.x; d < a.dim; d += 256)
      out[d] = from_f32<T>((f[0] * sums[0][d] + f[1] * sums[1][d] + f[2] * sums[2][d] + f[3] * sums[3][d]) * inv);
  }
}

// Joins a row's cuts, a wave a row.
template <typename T>
__global__ void __launch_bounds__(256) attend_any_join_kernel(AttendArgs a, int64_t rows) {
  const int lane = threadIdx.x & 63;
  const int64_t row = min((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), rows - 1);  // (the last row more than once)
  const int64_t token = (uint32_t)row / (uint32_t)a.q_heads;
  const int h = (int)(row - token * a.q_heads);
  if (sequence_of(a.seq, (int)token) < 0 && !a.zero_other) return;
  const float* part = a.part + row * a.splits * (a.dim + 2);
  const float factor = score_factor(a);
  float top = kNegInf, total = 0.0f;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, part[(int64_t)s * (a.dim + 2) + a.dim]);
  for (int s = 0; s < a.splits; ++s) {
    const float* x = part + (int64_t)s * (a.dim + 2) + a.dim;
    total += weight_of(x[0], top, factor) * x[1];
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  T* out = static_cast<T*>(a.out) + token * a.o_st + h * a.o_sh;
  for (int d = lane; d < a.dim; d += 64) {
    float sum = 0.0f;
    for (int s = 0; s < a.splits; ++s) {
      const float* x = part + (int64_t)s * (a.dim + 2);
      sum += weight_of(x[a.dim], top, factor) * x[d];
    }
    out[d] = from_f32<T>(sum * inv);
  }
}

// Cuts of a row's keys in the kernel above: workgroups for the whole GPU, each
// with 256 keys at least.
int any_splits(int64_t rows, int64_t max_keys) {
  const int64_t want = (1024 + rows - 1) / rows;
  return (int)std::max((int64_t)1, std::min({want, (int64_t)64, max_keys / 256}));
}

}  // namespace
}  // namespace ak

extern "C" size_t ak_paged_attention_workspace_bytes(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads,
                                                     int64_t dim, int64_t max_keys, int64_t max_chunk, int dtype) {
  if (tokens <= 0 || batch <= 0 || q_heads <= 0 || kv_heads <= 0 || dim <= 0 || max_keys < 0) return 0;
  max_chunk = std::max(max_chunk, (int64_t)1);
  // of the kernel that the call takes: by its pointers' alignment it may be either
  const int64_t rows = tokens * q_heads;
  const int splits = ak::any_splits(rows, max_keys);
  const size_t any = splits > 1 ? (size_t)(rows * splits * (dim + 2)) * sizeof(float) : 0;
  if (q_heads % kv_heads || dim > 256 || ak_dtype_size(dtype) == 0 || dim % (16 / ak_dtype_size(dtype))) return any;
  return std::max(any, ak::attend_tiles_workspace_bytes(tokens, batch, q_heads, kv_heads, dim, max_keys, max_chunk, dtype));
}

extern "C" int ak_paged_attention(const void* q, const void* k_cache, const void* v_cache, const int32_t* page_table,
                                  const int32_t* lengths, const int32_t* starts, void* out, void* workspace,
                                  size_t workspace_bytes, int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads,
                                  int64_t dim, int64_t n_pages, int64_t page_size, int64_t max_pages, int64_t ld_pages,
                                  int64_t max_chunk, int64_t q_st, int64_t q_sh, int64_t o_st, int64_t o_sh, int64_t kc_sp,
                                  int64_t kc_ss, int64_t kc_sh, int64_t vc_sp, int64_t vc_ss, int64_t vc_sh, float scale,
                                  float softcap, int64_t window, int flags, int dtype, void* stream) {
  const char* name = "ak_paged_attention";
  const int esz = ak_dtype_size(dtype);
  if (esz == 0) return ak_set_error(AK_ERR_UNSUPPORTED, "%s: unsupported dtype code %d", name, dtype);
  if (dim < 1 || dim > ak::kMaxAttendDim)
    return ak_set_error(AK_ERR_UNSUPPORTED, "%s: head dim %lld is not 1 to %lld", name, (long long)dim, (long long)ak::kMaxAttendDim);
  int rc = ak::check_paged(name, tokens, batch, n_pages, page_size, max_pages, ld_pages, starts, lengths, page_table);
  if (rc) return rc;
  if (q_heads < 1 || kv_heads < 1 || q_heads % kv_heads || q_heads > 65536 || tokens > INT32_MAX / q_heads ||
      (__int128)max_pages * page_size > INT32_MAX - 4096 || !ak::extent_ok(1, 0, tokens, q_st, q_heads, q_sh, dim, esz) ||
      !ak::extent_ok(1, 0, tokens, o_st, q_heads, o_sh, dim, esz) ||
      !ak::extent_ok(n_pages, kc_sp, page_size, kc_ss, kv_heads, kc_sh, dim, esz) ||
      !ak::extent_ok(n_pages, vc_sp, page_size, vc_ss, kv_heads, vc_sh, dim, esz))
    return ak_set_error(AK_ERR_INVALID_ARG, "%s: bad shape or strides", name);
  if (!(scale >= 1e-18f && scale <= 1e18f) || !(softcap == 0.0f || (softcap >= 1e-3f && softcap <= 1e4f)) || window < 0)
    return ak_set_error(AK_ERR_INVALID_ARG, "%s: scale must be 1e-18 to 1e18, softcap 0 or 1e-3 to 1e4, window not negative", name);
  if (tokens == 0) return AK_OK;
  if (!q || !out || (n_pages && (!k_cache || !v_cache))) return ak_set_error(AK_ERR_INVALID_ARG, "%s: null pointer", name);
  const int64_t max_keys = max_pages * page_size;
  const size_t need = ak_paged_attention_workspace_bytes(tokens, batch, q_heads, kv_heads, dim, max_keys, std::max(max_chunk, (int64_t)1), dtype);
  if (workspace_bytes < need || (need && (!workspace || !ak::aligned16(workspace))))
    return ak_set_error(AK_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed (16-byte aligned)", name, workspace_bytes, need);
  ak::AttendArgs a{};
  a.q = q;
  a.k = k_cache;
  a.v = v_cache;
  a.out = out;
  a.part = static_cast<float*>(workspace);
  a.seq = {starts, lengths, batch, tokens, starts ? 0 : tokens / batch};
  a.pages = page_table;
  a.n_pages = n_pages;
  a.page_size = page_size;
  a.max_pages = max_pages;
  a.ld_pages = ld_pages;
  a.q_st = q_st; a.q_sh = q_sh; a.o_st = o_st; a.o_sh = o_sh;
  a.kp = kc_sp; a.ks = kc_ss; a.kh = kc_sh; a.vp = vc_sp; a.vs = vc_ss; a.vh = vc_sh;
  a.window = window;
  a.q_heads = (int)q_heads;
  a.kv_heads = (int)kv_heads;
  a.dim = (int)dim;
  a.zero_other = (flags & AK_ZERO_OTHER_ROWS) != 0;
  a.scale = scale;
  a.softcap = softcap;
  hipStream_t s = ak_stream(stream);
  if (batch > 0 && ak::attend_tiles_take(a, dtype)) {
    ak::attend_tiles(a, std::max(max_chunk, (int64_t)1), dtype, workspace, s);
    return ak_check_launch(name);
  }
  const int64_t rows = tokens * q_heads;
  a.splits = batch > 0 ? ak::any_splits(rows, max_keys) : 1;
  auto go = [&](auto t) {
    using T = decltype(t);
    ak::attend_any_kernel<T><<<dim3(ak::row_grid(rows), (unsigned)a.splits), dim3(256), 0, s>>>(a, rows);
    if (a.splits > 1) ak::attend_any_join_kernel<T><<<dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s>>>(a, rows);
  };
  if (dtype == AK_DTYPE_F32) go(float());
  else if (dtype == AK_DTYPE_F16) go(ak::f16());
  else go(ak::bf16());
  return ak_check_launch(name);
}
