// Attention of new tokens over a paged key-value cache.
//
// One block per query and head: its warps take the keys in turn with a running maximum and sum each and are joined at the end.
#include <cuda_bf16.h>

#include <cmath>

#include "paged_cache.h"

namespace tf {

struct AttendArgs {
  tf_paged_cache cache;
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  float* lse;
  int64_t q_ldt, q_ldh, out_ldt, out_ldh;
  const int32_t* tables;
  int64_t table_cols, table_stride;
  const int32_t* lengths;
  const int32_t* counts;
  int queries, q_heads, group, d;
  float scale_log2;
  int64_t window;
};

constexpr int kAttendWarps = 4;

__device__ __forceinline__ float entry_value(const void* base, int64_t at, bool codes) {
  return codes ? e4m3_to_f32(static_cast<const uint8_t*>(base)[at]) : __bfloat162float(static_cast<const __nv_bfloat16*>(base)[at]);
}

__global__ void __launch_bounds__(32 * kAttendWarps) paged_attention_kernel(AttendArgs p) {
  const int64_t token = blockIdx.x;
  const int head = blockIdx.y, kv = head / p.group, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t b = token / p.queries;
  const int i = (int)(token - b * p.queries);
  const int64_t cap = p.table_cols * p.cache.page_size;
  int64_t len = p.lengths[b];
  len = len < 0 ? 0 : len > cap ? cap : len;
  int n = p.counts ? p.counts[b] : p.queries;
  n = n < 0 ? 0 : n > p.queries ? p.queries : n;
  const int64_t end = i < n ? len - n + 1 + i : 0, begin = p.window && end > p.window ? end - p.window : 0;
  const bool codes = p.cache.dtype == TF_CACHE_E4M3;
  const __nv_bfloat16* q = p.q + token * p.q_ldt + head * p.q_ldh;
  float qv[8], o[8], m = -INFINITY, l = 0.0f;
  const float ks = codes && p.cache.k_scale ? load_f32(p.cache.k_scale + kv) : 1.0f;
  for (int j = 0; j < 8; ++j) {
    qv[j] = lane + 32 * j < p.d ? __bfloat162float(q[lane + 32 * j]) : 0.0f;
    o[j] = 0.0f;
  }
  for (int64_t e = begin + warp; e < end; e += kAttendWarps) {
    const int64_t col = e / p.cache.page_size;
    const int32_t page = p.tables[b * p.table_stride + col];
    if (page < 0 || page >= p.cache.pages) continue;
    const int64_t at = page * p.cache.stride_page + kv * p.cache.stride_head + (e - col * p.cache.page_size) * p.cache.stride_slot;
    float s = 0.0f;
    for (int j = 0; j < 8; ++j)
      if (lane + 32 * j < p.d) s = fmaf(qv[j], entry_value(p.cache.k, at + lane + 32 * j, codes), s);
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(~0u, s, x);
    s *= p.scale_log2 * ks;
    const float top = fmaxf(m, s), base = top == -INFINITY ? 0.0f : top, keep = exp2f(m - base), w = exp2f(s - base);
    m = top;
    l = l * keep + w;
    for (int j = 0; j < 8; ++j)
      if (lane + 32 * j < p.d) o[j] = fmaf(w, entry_value(p.cache.v, at + lane + 32 * j, codes), o[j] * keep);
  }
  __shared__ float so[kAttendWarps][256], sm[kAttendWarps], sl[kAttendWarps];
  for (int j = 0; j < 8; ++j) so[warp][lane + 32 * j] = o[j];
  if (lane == 0) sm[warp] = m, sl[warp] = l;
  __syncthreads();
  float top = -INFINITY, sum = 0.0f, w[kAttendWarps];
  for (int x = 0; x < kAttendWarps; ++x) top = fmaxf(top, sm[x]);
  const float base = top == -INFINITY ? 0.0f : top;
  for (int x = 0; x < kAttendWarps; ++x) {
    w[x] = exp2f(sm[x] - base);
    sum += w[x] * sl[x];
  }
  const float vs = (codes && p.cache.v_scale ? load_f32(p.cache.v_scale + kv) : 1.0f);
  for (int c = threadIdx.x; c < p.d; c += blockDim.x) {
    float x = 0.0f;
    for (int y = 0; y < kAttendWarps; ++y) x += w[y] * so[y][c];
    p.out[token * p.out_ldt + head * p.out_ldh + c] = __float2bfloat16_rn(sum == 0.0f ? 0.0f : x / sum * vs);
  }
  if (threadIdx.x == 0 && p.lse) p.lse[token * p.q_heads + head] = sum == 0.0f ? -INFINITY : (base + log2f(sum)) * 0.6931471805599453f;
}

}  // namespace tf

using namespace tf;

extern "C" int64_t tf_paged_attention_workspace_bytes(int64_t seqs, int64_t queries, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int32_t cache_dtype,
                                                      int64_t max_entries) {
  return seqs < 0 || queries < 1 || q_heads < 1 || kv_heads < 1 || head_dim < 16 || max_entries < 1 || cache_dtype < 0 || cache_dtype > 1 ? -1 : 0;
}

extern "C" tf_status tf_paged_attention(const tf_paged_cache* cache, const void* q, int64_t q_stride_token, int64_t q_stride_head, int64_t seqs, int64_t queries,
                                        int64_t q_heads, const int32_t* tables, int64_t table_cols, int64_t table_stride, const int32_t* lengths,
                                        const int32_t* counts, float scale, int64_t window, void* out, int64_t out_stride_token, int64_t out_stride_head,
                                        float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  if (tf_status st = check_cache(cache, __func__)) return st;
  TF_CHECK_ARG(q && out && tables && lengths, "%s: null pointer", __func__);
  TF_CHECK_ARG(seqs >= 0 && queries > 0 && q_heads > 0 && seqs * queries <= INT32_MAX && q_heads <= 65535 && table_cols > 0 && window >= 0,
               "%s: bad shape seqs=%lld queries=%lld q_heads=%lld table_cols=%lld window=%lld", __func__, (long long)seqs, (long long)queries, (long long)q_heads,
               (long long)table_cols, (long long)window);
  TF_CHECK_ARG(q_heads % cache->kv_heads == 0, "%s: q_heads=%lld is not a multiple of kv_heads=%lld", __func__, (long long)q_heads, (long long)cache->kv_heads);
  TF_CHECK_ALIGNED(q, 16, "q");
  TF_CHECK_ALIGNED(out, 16, "out");
  TF_CHECK_ALIGNED(workspace, 16, "workspace");
  if (q_stride_token % 8 || q_stride_head % 8 || out_stride_token % 8 || out_stride_head % 8)
    return fail(TF_ERR_ALIGNMENT, "%s: the strides must be multiples of 8 elements", __func__);
  if (seqs == 0) return TF_OK;
  AttendArgs p = {};
  p.cache = *cache;
  p.q = static_cast<const __nv_bfloat16*>(q), p.out = static_cast<__nv_bfloat16*>(out), p.lse = lse;
  p.q_ldt = q_stride_token, p.q_ldh = q_stride_head, p.out_ldt = out_stride_token, p.out_ldh = out_stride_head;
  p.tables = tables, p.table_cols = table_cols, p.table_stride = table_stride, p.lengths = lengths, p.counts = counts;
  p.queries = (int)queries, p.q_heads = (int)q_heads, p.group = (int)(q_heads / cache->kv_heads), p.d = (int)cache->head_dim;
  p.scale_log2 = scale * 1.4426950408889634f, p.window = window;
  (void)workspace_bytes;
  paged_attention_kernel<<<dim3((unsigned)(seqs * queries), (unsigned)q_heads), 32 * kAttendWarps, 0, (cudaStream_t)stream>>>(p);
  TF_LAUNCH_CHECK();
  return TF_OK;
}
