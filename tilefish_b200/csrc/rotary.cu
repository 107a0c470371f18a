// Rotary positions, alone and on the way into a paged key-value cache: checks and entry points.
#include "rotary.cuh"

namespace tf {

static tf_status check_rotation(const uint64_t* turns, int64_t rot, int64_t d, int32_t layout, int32_t position_bits, const char* fn) {
  if (position_bits != 32 && position_bits != 64) return fail(TF_ERR_INVALID_ARGUMENT, "%s: position_bits is 32 or 64", fn);
  if (layout != TF_ROTARY_HALF && layout != TF_ROTARY_INTERLEAVED) return fail(TF_ERR_INVALID_ARGUMENT, "%s: unknown layout %d", fn, layout);
  if (rot < 0 || rot % 2 || rot > d || (rot > 0) != (turns != nullptr))
    return fail(TF_ERR_INVALID_ARGUMENT, "%s: rot=%lld must be even, at most head_dim=%lld, and come with turns", fn, (long long)rot, (long long)d);
  if (reinterpret_cast<uintptr_t>(turns) % 8) return fail(TF_ERR_ALIGNMENT, "%s: turns must be 8-byte aligned", fn);
  return TF_OK;
}

}  // namespace tf

using namespace tf;

extern "C" tf_status tf_rotary(const void* x, int32_t dtype, int64_t tokens, int64_t heads, int64_t head_dim, int64_t x_stride_token, int64_t x_stride_head,
                               const void* positions, int32_t position_bits, const uint64_t* turns, int64_t rot, int32_t layout, float magnitude,
                               int32_t inverse, void* out, int64_t out_stride_token, int64_t out_stride_head, void* stream) {
  clear_error();
  TF_CHECK_ARG(x && out && positions && turns, "%s: null pointer", __func__);
  TF_CHECK_ARG(dtype == TF_BF16 || dtype == TF_F32, "%s: unknown dtype %d", __func__, dtype);
  TF_CHECK_ARG(tokens >= 0 && tokens < (1ll << 40) && heads > 0 && heads <= 65535 && head_dim > 0 && head_dim <= 1024, "%s: bad shape tokens=%lld heads=%lld head_dim=%lld", __func__,
               (long long)tokens, (long long)heads, (long long)head_dim);
  if (tf_status st = check_rotation(turns, rot, head_dim, layout, position_bits, __func__)) return st;
  const int64_t item = dtype == TF_BF16 ? 2 : 4;
  TF_CHECK_ALIGNED(x, item, "x");
  TF_CHECK_ALIGNED(out, item, "out");
  TF_CHECK_ALIGNED(positions, position_bits / 8, "positions");
  if (tokens == 0) return TF_OK;
  RotaryArgs p = {};
  p.q = x, p.q_ldt = x_stride_token, p.q_ldh = x_stride_head;
  p.q_out = out, p.qo_ldt = out_stride_token, p.qo_ldh = out_stride_head;
  p.positions = positions, p.wide_positions = position_bits == 64;
  p.turns = turns, p.magnitude = magnitude, p.inverse = inverse != 0, p.interleaved = layout == TF_ROTARY_INTERLEAVED;
  p.tokens = tokens, p.q_heads = p.heads = (int)heads, p.d = (int)head_dim, p.rot = (int)rot;
  p.in_place = x == out;
  return dtype == TF_BF16 ? launch_rotary<__nv_bfloat16>(p, (cudaStream_t)stream) : launch_rotary<float>(p, (cudaStream_t)stream);
}

extern "C" tf_status tf_cache_append(const tf_paged_cache* cache, const void* k, int64_t k_stride_token, int64_t k_stride_head, const void* v,
                                     int64_t v_stride_token, int64_t v_stride_head, int64_t tokens, const int32_t* tables, int64_t table_rows,
                                     int64_t table_cols, int64_t table_stride, const void* positions, int32_t position_bits, const int32_t* rows, const void* q,
                                     int64_t q_heads, int64_t q_stride_token, int64_t q_stride_head, void* q_out, int64_t q_out_stride_token,
                                     int64_t q_out_stride_head, const uint64_t* turns, int64_t rot, int32_t layout, float magnitude, void* stream) {
  clear_error();
  if (tf_status st = check_cache(cache, __func__)) return st;
  TF_CHECK_ARG(k && v && tables && positions && (q != nullptr) == (q_out != nullptr), "%s: null pointer", __func__);
  TF_CHECK_ARG(tokens >= 0 && tokens < (1ll << 40) && table_rows > 0 && table_cols > 0 && q_heads >= 0 && q_heads <= 65535 && (q_heads > 0) == (q != nullptr),
               "%s: bad shape tokens=%lld table=[%lld, %lld] q_heads=%lld", __func__, (long long)tokens, (long long)table_rows, (long long)table_cols,
               (long long)q_heads);
  TF_CHECK_ARG(rows || tokens % table_rows == 0, "%s: without rows, tokens=%lld must be a multiple of the table's %lld rows", __func__, (long long)tokens,
               (long long)table_rows);
  if (tf_status st = check_rotation(turns, rot, cache->head_dim, layout, position_bits, __func__)) return st;
  TF_CHECK_ALIGNED(k, 16, "k");
  TF_CHECK_ALIGNED(v, 16, "v");
  TF_CHECK_ALIGNED(q, 16, "q");
  TF_CHECK_ALIGNED(q_out, 16, "q_out");
  TF_CHECK_ALIGNED(tables, 4, "tables");
  TF_CHECK_ALIGNED(rows, 4, "rows");
  TF_CHECK_ALIGNED(positions, position_bits / 8, "positions");
  if (k_stride_token % 8 || k_stride_head % 8 || v_stride_token % 8 || v_stride_head % 8 || q_stride_token % 8 || q_stride_head % 8 || q_out_stride_token % 8 ||
      q_out_stride_head % 8)
    return fail(TF_ERR_ALIGNMENT, "%s: the strides must be multiples of 8 elements", __func__);
  if (tokens == 0) return TF_OK;
  RotaryArgs p = {};
  p.q = q, p.q_ldt = q_stride_token, p.q_ldh = q_stride_head;
  p.q_out = q_out, p.qo_ldt = q_out_stride_token, p.qo_ldh = q_out_stride_head;
  p.k = static_cast<const __nv_bfloat16*>(k), p.k_ldt = k_stride_token, p.k_ldh = k_stride_head;
  p.v = static_cast<const __nv_bfloat16*>(v), p.v_ldt = v_stride_token, p.v_ldh = v_stride_head;
  p.cache = *cache;
  // no sequence has more than 2^30 entries
  const int64_t most = INT32_MAX / 2, page = cache->page_size > most ? most : cache->page_size;
  p.tables = tables, p.table_rows = table_rows, p.table_stride = table_stride;
  p.entries = (int)(table_cols > most / page ? most : table_cols * page), p.page = divisor((int)page);
  p.rows = rows, p.tokens_per_row = rows ? 1 : tokens / table_rows;
  p.positions = positions, p.wide_positions = position_bits == 64;
  p.turns = turns, p.magnitude = magnitude, p.interleaved = layout == TF_ROTARY_INTERLEAVED;
  p.tokens = tokens, p.q_heads = (int)q_heads, p.heads = (int)(q_heads + 2 * cache->kv_heads), p.d = (int)cache->head_dim, p.rot = (int)rot;
  p.in_place = q == q_out;
  return launch_rotary_vectors<__nv_bfloat16, true>(p, (cudaStream_t)stream);
}
