// The entry points of attention over a paged key-value cache. The kernels are in paged_attention.cuh, built by head size in paged_attention_<type>_d<size>.cu.
#include <cmath>
#include <type_traits>

#include "paged_attention.h"

namespace tf {

extern template struct AttendCall<64, false, 8>;
extern template struct AttendCall<64, false, 16>;
extern template struct AttendCall<64, false, 24>;
extern template struct AttendCall<64, false, 32>;
extern template struct AttendCall<64, false, 48>;
extern template struct AttendCall<64, false, 64>;
extern template struct AttendCall<64, true, 8>;
extern template struct AttendCall<64, true, 16>;
extern template struct AttendCall<64, true, 24>;
extern template struct AttendCall<64, true, 32>;
extern template struct AttendCall<64, true, 48>;
extern template struct AttendCall<64, true, 64>;
extern template struct AttendCall<96, false, 8>;
extern template struct AttendCall<96, false, 16>;
extern template struct AttendCall<96, false, 24>;
extern template struct AttendCall<96, false, 32>;
extern template struct AttendCall<96, false, 48>;
extern template struct AttendCall<96, false, 64>;
extern template struct AttendCall<96, true, 8>;
extern template struct AttendCall<96, true, 16>;
extern template struct AttendCall<96, true, 24>;
extern template struct AttendCall<96, true, 32>;
extern template struct AttendCall<96, true, 48>;
extern template struct AttendCall<96, true, 64>;
extern template struct AttendCall<128, false, 8>;
extern template struct AttendCall<128, false, 16>;
extern template struct AttendCall<128, false, 24>;
extern template struct AttendCall<128, false, 32>;
extern template struct AttendCall<128, false, 48>;
extern template struct AttendCall<128, false, 64>;
extern template struct AttendCall<128, true, 8>;
extern template struct AttendCall<128, true, 16>;
extern template struct AttendCall<128, true, 24>;
extern template struct AttendCall<128, true, 32>;
extern template struct AttendCall<128, true, 48>;
extern template struct AttendCall<128, true, 64>;
extern template struct AttendCall<256, false, 8>;
extern template struct AttendCall<256, false, 16>;
extern template struct AttendCall<256, false, 32>;
extern template struct AttendCall<256, false, 64>;
extern template struct AttendCall<256, true, 8>;
extern template struct AttendCall<256, true, 16>;
extern template struct AttendCall<256, true, 32>;
extern template struct AttendCall<256, true, 64>;

// Rows of a tile: as few as hold a kv head's query heads times the new tokens, up to 64; more are several tiles, which read the keys again. One tile is faster
// than several small ones (12 sequences of up to 16384, bf16: 64 rows of 128 elements 112 us, in tiles of 24 and 16 137 and 181; 48 of 96 elements 67, 84 and 94)
// but for 33 to 48 rows of more than 128 elements, for which 64 is a third too many (256 elements: 284 us, in tiles of 16 270; e4m3 169 and 143).
static int attend_rows(int64_t rows, int64_t d) {
  const int64_t tiles = (rows + 63) / 64;
  rows = (rows + tiles - 1) / tiles;  // 80 are twice 40
  if (d > 128) return rows <= 8 ? 8 : rows <= 16 || (rows > 32 && rows <= 48) ? 16 : rows <= 32 ? 32 : 64;
  const int eights = (int)(rows + 7) / 8;
  return eights <= 4 ? 8 * eights : eights <= 6 ? 48 : 64;
}
static int64_t attend_row_tiles(int64_t rows, int64_t d) {
  const int tile = attend_rows(rows, d);
  return (rows + tile - 1) / tile;
}

template <class Use>
static auto with_attend_call(int64_t rows, int64_t d, int32_t dtype, Use use) {
  auto by_rows = [&](auto dp, auto f8) {
    constexpr int kDP = decltype(dp)::value;
    constexpr bool kF8 = decltype(f8)::value;
    const int tile = attend_rows(rows, d);
    if (tile == 8) return use(AttendCall<kDP, kF8, 8>{});
    if (tile == 16) return use(AttendCall<kDP, kF8, 16>{});
    if (tile == 32) return use(AttendCall<kDP, kF8, 32>{});
    if constexpr (kDP < 256) {
      if (tile == 24) return use(AttendCall<kDP, kF8, 24>{});
      if (tile == 48) return use(AttendCall<kDP, kF8, 48>{});
    }
    return use(AttendCall<kDP, kF8, 64>{});
  };
  auto by_dim = [&](auto f8) {
    return d <= 64 ? by_rows(std::integral_constant<int, 64>{}, f8) : d <= 96 ? by_rows(std::integral_constant<int, 96>{}, f8) : d <= 128 ? by_rows(std::integral_constant<int, 128>{}, f8) : by_rows(std::integral_constant<int, 256>{}, f8);
  };
  return dtype == TF_CACHE_E4M3 ? by_dim(std::true_type{}) : by_dim(std::false_type{});
}

// Sizes that the kernels' 32-bit counts hold.
static bool attend_sizes_ok(int64_t seqs, int64_t queries, int64_t q_heads, int64_t kv_heads, int64_t d) {
  if (seqs < 0 || queries < 1 || q_heads < 1 || kv_heads < 1 || kv_heads > 65535 || q_heads > 65535 || q_heads % kv_heads) return false;
  if (seqs > (1 << 30) || queries > (1 << 20)) return false;
  const int64_t rows = queries * (q_heads / kv_heads);
  return rows < (1 << 30) && seqs * queries <= INT32_MAX && seqs * attend_row_tiles(rows, d) * kv_heads <= INT32_MAX;
}

}  // namespace tf

using namespace tf;

extern "C" int64_t tf_paged_attention_workspace_bytes(int64_t seqs, int64_t queries, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int32_t cache_dtype,
                                                      int64_t max_entries) {
  if (!attend_sizes_ok(seqs, queries, q_heads, kv_heads, head_dim) || head_dim < 16 || head_dim > 256 || head_dim % 16 || max_entries < 1 || cache_dtype < 0 || cache_dtype > 1) return -1;
  const int64_t rows = queries * (q_heads / kv_heads), entries = max_entries > INT32_MAX / 2 ? INT32_MAX / 2 : max_entries;
  if (seqs == 0) return 0;
  return with_attend_call(rows, head_dim, cache_dtype, [&](auto call) { return decltype(call)::workspace(seqs * attend_row_tiles(rows, head_dim), kv_heads, entries); });
}

extern "C" tf_status tf_paged_attention(const tf_paged_cache* cache, const void* q, int64_t q_stride_token, int64_t q_stride_head, int64_t seqs, int64_t queries,
                                        int64_t q_heads, const int32_t* tables, int64_t table_cols, int64_t table_stride, const int32_t* lengths,
                                        const int32_t* counts, float scale, int64_t window, void* out, int64_t out_stride_token, int64_t out_stride_head,
                                        float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  if (tf_status st = check_cache(cache, __func__)) return st;
  TF_CHECK_ARG(q && out && tables && lengths, "%s: null pointer", __func__);
  TF_CHECK_ARG(attend_sizes_ok(seqs, queries, q_heads, cache->kv_heads, cache->head_dim) && table_cols > 0 && window >= 0,
               "%s: bad shape seqs=%lld queries=%lld q_heads=%lld kv_heads=%lld table_cols=%lld window=%lld", __func__, (long long)seqs, (long long)queries,
               (long long)q_heads, (long long)cache->kv_heads, (long long)table_cols, (long long)window);
  TF_CHECK_ALIGNED(q, 16, "q");
  TF_CHECK_ALIGNED(out, 16, "out");
  TF_CHECK_ALIGNED(workspace, 16, "workspace");
  TF_CHECK_ALIGNED(tables, 4, "tables");
  TF_CHECK_ALIGNED(lengths, 4, "lengths");
  TF_CHECK_ALIGNED(counts, 4, "counts");
  TF_CHECK_ALIGNED(lse, 4, "lse");
  TF_CHECK_ARG(std::isfinite(scale), "%s: scale is not finite", __func__);
  if (q_stride_token % 8 || q_stride_head % 8 || out_stride_token % 8 || out_stride_head % 8)
    return fail(TF_ERR_ALIGNMENT, "%s: the strides must be multiples of 8 elements", __func__);
  if (seqs == 0) return TF_OK;
  // a table that names more entries than 2^30 is read up to there: no sequence is that long
  const int64_t most = INT32_MAX / 2, entries = table_cols > most / cache->page_size ? most : table_cols * cache->page_size;
  const int64_t item = cache->dtype == TF_CACHE_BF16 ? 2 : 1, rows = queries * (q_heads / cache->kv_heads);
  AttendArgs p = {};
  p.k = static_cast<const uint8_t*>(cache->k), p.v = static_cast<const uint8_t*>(cache->v), p.k_scale = cache->k_scale, p.v_scale = cache->v_scale;
  p.stride_page = cache->stride_page * item, p.stride_head = cache->stride_head * item, p.stride_slot = cache->stride_slot * item;
  p.pages = (int)cache->pages, p.kv_heads = (int)cache->kv_heads, p.d = (int)cache->head_dim;
  p.page = divisor((int)(cache->page_size > most ? most : cache->page_size));
  p.q = static_cast<const __nv_bfloat16*>(q), p.out = static_cast<__nv_bfloat16*>(out), p.lse = lse;
  p.q_ldt = q_stride_token, p.q_ldh = q_stride_head, p.out_ldt = out_stride_token, p.out_ldh = out_stride_head;
  p.tables = tables, p.table_stride = table_stride, p.lengths = lengths, p.counts = counts, p.entries = (int)entries;
  p.queries = (int)queries, p.q_heads = (int)q_heads, p.row_tiles = (int)attend_row_tiles(rows, cache->head_dim), p.spans = (int)(seqs * p.row_tiles);
  p.window = (int)(window > INT32_MAX / 2 ? 0 : window);
  p.group = divisor((int)(q_heads / cache->kv_heads));
  p.scale_log2 = scale * 1.4426950408889634f;
  return with_attend_call(rows, p.d, cache->dtype, [&](auto call) { return decltype(call)::launch(p, workspace, workspace_bytes, (cudaStream_t)stream, "tf_paged_attention"); });
}
