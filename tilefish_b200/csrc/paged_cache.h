// What the rotary and paged-attention kernels share: the check of a cache's descriptor, and a division.
#pragma once

#include "common.cuh"

namespace tf {

inline tf_status check_cache(const tf_paged_cache* c, const char* fn) {
  if (!c || !c->k || !c->v) return fail(TF_ERR_INVALID_ARGUMENT, "%s: null cache", fn);
  if (c->dtype != TF_CACHE_BF16 && c->dtype != TF_CACHE_E4M3) return fail(TF_ERR_INVALID_ARGUMENT, "%s: unknown cache dtype %d", fn, c->dtype);
  if (c->pages < 1 || c->pages > INT32_MAX || c->page_size < 1 || c->page_size > INT32_MAX || c->kv_heads < 1 || c->kv_heads > 65535)
    return fail(TF_ERR_INVALID_ARGUMENT, "%s: bad cache shape (pages %lld, page_size %lld, kv_heads %lld)", fn, (long long)c->pages, (long long)c->page_size,
                (long long)c->kv_heads);
  if (c->head_dim < 16 || c->head_dim > 256 || c->head_dim % 16)
    return fail(TF_ERR_UNSUPPORTED, "%s: head_dim %lld is not a multiple of 16 up to 256", fn, (long long)c->head_dim);
  const int64_t unit = c->dtype == TF_CACHE_BF16 ? 8 : 16;
  if (c->stride_page % unit || c->stride_head % unit || c->stride_slot % unit || c->stride_page < 0 || c->stride_head < 0 || c->stride_slot < 0)
    return fail(TF_ERR_ALIGNMENT, "%s: the cache's strides must be multiples of 16 bytes", fn);
  if (reinterpret_cast<uintptr_t>(c->k) % 16 || reinterpret_cast<uintptr_t>(c->v) % 16) return fail(TF_ERR_ALIGNMENT, "%s: k and v must be 16-byte aligned", fn);
  if (reinterpret_cast<uintptr_t>(c->k_scale) % 4 || reinterpret_cast<uintptr_t>(c->v_scale) % 4) return fail(TF_ERR_ALIGNMENT, "%s: the scales must be 4-byte aligned", fn);
  if (c->dtype == TF_CACHE_BF16 && (c->k_scale || c->v_scale)) return fail(TF_ERR_INVALID_ARGUMENT, "%s: a bf16 cache has no scales", fn);
  return TF_OK;
}

// floor(n / d) for 0 <= n < 2^31 by a multiplication: with 2^l >= d, m = ceil(2^(31 + l) / d) exceeds the quotient by less than 2^l / d parts.
struct Divisor {
  uint32_t mul, shift;
  int d;
};
inline Divisor divisor(int d) {
  int l = 0;
  while ((1ll << l) < d) ++l;
  return {(uint32_t)(((1ull << (31 + l)) + d - 1) / d), (uint32_t)(31 + l), d};
}
#ifdef __CUDACC__
__device__ __forceinline__ int divide(int n, Divisor v) { return (int)(((uint64_t)(uint32_t)n * v.mul) >> v.shift); }
#endif

}  // namespace tf
