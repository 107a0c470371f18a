// Rotary positions, alone (tf_rotary) and on the way into a paged key-value cache (tf_cache_append).
//
// Pair i of a head of token t becomes (a c - b s, b c + a s) with c = m cos(theta), s = m sin(theta), theta = positions[t] * f_i. The angle is
// kept as the fraction of a turn in 64-bit fixed point, turns_i = f_i / 2 pi * 2^64: the product with the position wraps modulo a whole turn
// by itself, so its error is |position| * 2^-65 turns at any position (an f32 product is off by a tenth of a radian at position one million).
// The upper 32 bits go to sincospif as an argument in [-1, 1).
#include <cuda_bf16.h>

#include "paged_cache.h"

namespace tf {

struct RotaryArgs {
  // queries (or the one tensor of tf_rotary): heads [0, q_heads) of a token
  const void* q;
  void* q_out;
  int64_t q_ldt, q_ldh, qo_ldt, qo_ldh;
  // keys and values: the next kv_heads and the last kv_heads
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  int64_t k_ldt, k_ldh, v_ldt, v_ldh;
  tf_paged_cache cache;
  const int32_t* tables;
  int64_t table_rows, table_cols, table_stride;
  const int32_t* rows;
  int64_t tokens_per_row;
  const void* positions;
  const uint64_t* turns;
  float magnitude;
  int64_t tokens;
  int q_heads, heads;  // heads: of all three
  int d, rot;
  bool wide_positions, interleaved, inverse, in_place;
};

constexpr int kRotaryThreads = 256;

__device__ __forceinline__ int64_t position_of(const RotaryArgs& p, int64_t t) {
  return p.wide_positions ? reinterpret_cast<const int64_t*>(p.positions)[t] : (int64_t) reinterpret_cast<const int32_t*>(p.positions)[t];
}

__device__ __forceinline__ float2 cos_sin(const RotaryArgs& p, int64_t position, int pair) {
  const uint64_t turn = (uint64_t)position * p.turns[pair];
  const float half_turns = (float)(int32_t)((turn + 0x80000000ull) >> 32) * 0x1p-31f;
  float s, c;
  sincospif(half_turns, &s, &c);
  return make_float2(c * p.magnitude, (p.inverse ? -s : s) * p.magnitude);
}

// Where the key or value of token t goes: its byte offset in the cache's k or v, or -1 where nothing is written.
__device__ __forceinline__ int64_t entry_offset(const RotaryArgs& p, int64_t t, int head) {
  const int64_t e = position_of(p, t);
  const int64_t row = p.rows ? (int64_t)p.rows[t] : t / p.tokens_per_row;
  if (e < 0 || row < 0 || row >= p.table_rows) return -1;
  const int64_t col = e / p.cache.page_size;
  if (col >= p.table_cols) return -1;
  const int32_t page = p.tables[row * p.table_stride + col];
  if (page < 0 || page >= p.cache.pages) return -1;
  const int64_t at = page * p.cache.stride_page + head * p.cache.stride_head + (e - col * p.cache.page_size) * p.cache.stride_slot;
  return p.cache.dtype == TF_CACHE_BF16 ? at * 2 : at;
}

__device__ __forceinline__ float as_f32(float x) { return x; }
__device__ __forceinline__ float as_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* to, float x) { *to = x; }
__device__ __forceinline__ void put(__nv_bfloat16* to, float x) { *to = __float2bfloat16_rn(x); }

// One element or pair per thread: any even rot, any alignment.
template <typename T, bool kAppend>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(RotaryArgs p) {
  const int half = p.rot / 2, items = half + (p.d - p.rot);
  const int64_t total = p.tokens * p.heads * items;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / items;
    const int item = (int)(i - row * items);
    const int64_t t = row / p.heads;
    const int head = (int)(row - t * p.heads);
    const T* src;
    T* dst = nullptr;
    uint8_t* code = nullptr;
    float inv_scale = 1.0f;
    bool turned = true;
    if (!kAppend || head < p.q_heads) {
      src = reinterpret_cast<const T*>(p.q) + t * p.q_ldt + head * p.q_ldh;
      dst = reinterpret_cast<T*>(p.q_out) + t * p.qo_ldt + head * p.qo_ldh;
    } else {
      const int kv = (int)p.cache.kv_heads;
      const bool key = head < p.q_heads + kv;
      const int h = head - p.q_heads - (key ? 0 : kv);
      const int64_t at = entry_offset(p, t, h);
      if (at < 0) continue;
      src = reinterpret_cast<const T*>(key ? p.k + t * p.k_ldt + h * p.k_ldh : p.v + t * p.v_ldt + h * p.v_ldh);
      uint8_t* entry = static_cast<uint8_t*>(key ? p.cache.k : p.cache.v) + at;
      if (p.cache.dtype == TF_CACHE_BF16) {
        dst = reinterpret_cast<T*>(entry);
      } else {
        code = entry;
        const float* scale = key ? p.cache.k_scale : p.cache.v_scale;
        if (scale) inv_scale = __frcp_rn(load_f32(scale + h));
      }
      turned = key;
    }
    if (item < half) {
      const int i0 = p.interleaved ? 2 * item : item, i1 = p.interleaved ? 2 * item + 1 : item + half;
      float a = as_f32(src[i0]), b = as_f32(src[i1]);
      if (!turned && !code) {  // a copy keeps its bits
        dst[i0] = src[i0];
        dst[i1] = src[i1];
        continue;
      }
      if (turned) {
        const float2 cs = cos_sin(p, position_of(p, t), item);
        const float x = fmaf(a, cs.x, -(b * cs.y)), y = fmaf(b, cs.x, a * cs.y);
        a = x;
        b = y;
      }
      if (code) {
        const uint32_t two = cvt_e4m3x2(a * inv_scale, b * inv_scale);
        code[i0] = (uint8_t)two;
        code[i1] = (uint8_t)(two >> 8);
      } else {
        put(dst + i0, a);
        put(dst + i1, b);
      }
    } else {
      const int e = p.rot + item - half;
      if (code)
        code[e] = (uint8_t)cvt_e4m3x2(as_f32(src[e]) * inv_scale, 0.0f);
      else
        dst[e] = src[e];
    }
  }
}

template <typename T, bool kAppend>
static tf_status launch_rotary(const RotaryArgs& p, cudaStream_t stream) {
  const int64_t total = p.tokens * p.heads * (p.d - p.rot / 2), cap = (int64_t)sm_count() * 8;
  const int64_t need = (total + kRotaryThreads - 1) / kRotaryThreads;
  rotary_kernel<T, kAppend><<<(unsigned)(need < cap ? need : cap), kRotaryThreads, 0, stream>>>(p);
  TF_LAUNCH_CHECK();
  return TF_OK;
}

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
  return dtype == TF_BF16 ? launch_rotary<__nv_bfloat16, false>(p, (cudaStream_t)stream) : launch_rotary<float, false>(p, (cudaStream_t)stream);
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
  p.tables = tables, p.table_rows = table_rows, p.table_cols = table_cols, p.table_stride = table_stride;
  p.rows = rows, p.tokens_per_row = rows ? 1 : tokens / table_rows;
  p.positions = positions, p.wide_positions = position_bits == 64;
  p.turns = turns, p.magnitude = magnitude, p.interleaved = layout == TF_ROTARY_INTERLEAVED;
  p.tokens = tokens, p.q_heads = (int)q_heads, p.heads = (int)(q_heads + 2 * cache->kv_heads), p.d = (int)cache->head_dim, p.rot = (int)rot;
  p.in_place = q == q_out;
  return launch_rotary<__nv_bfloat16, true>(p, (cudaStream_t)stream);
}
