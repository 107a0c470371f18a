// Kernels of rotary positions, alone (tf_rotary) and on the way into a paged key-value cache (tf_cache_append), and their launches.
//
// Pair i of a head of token t becomes (a c - b s, b c + a s) with c = m cos(theta), s = m sin(theta), theta = positions[t] * f_i. The angle is
// kept as the fraction of a turn in 64-bit fixed point, turns_i = f_i / 2 pi * 2^64: the product with the position wraps modulo a whole turn
// by itself, so its error is |position| * 2^-65 turns at any position (an f32 product is off by a tenth of a radian at position one million).
// The nearest quarter turn is taken off as an integer; what is left, at most an eighth of a turn, goes to sincospif rounded to f32: 2^-28 turns at
// the most, and cosines and sines near zero keep their relative accuracy (the whole turn rounded to f32 was off by up to 2^-26 turns; one head of 8192 tokens
// 4.4 us so, 4.8 now in f32, 64 heads 40.8 either way).
#pragma once
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
  int64_t table_rows, table_stride;
  int entries;  // what a table can name
  Divisor page;
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
  const uint32_t quarter = (uint32_t)((turn + (1ull << 61)) >> 62);
  const int64_t left = (int64_t)(turn - ((uint64_t)quarter << 62));
  float s, c;
  sincospif((float)left * 0x1p-63f, &s, &c);
  const float x = quarter & 1 ? s : c, y = quarter & 1 ? c : s;
  return make_float2(((quarter + 1) & 2 ? -x : x) * p.magnitude, (((quarter >> 1) != 0) != p.inverse ? -y : y) * p.magnitude);
}

// Where the key and value of token t go: byte offset of the first head's in the cache's k and v, or -1 where nothing is written.
__device__ __forceinline__ int64_t entry_offset(const RotaryArgs& p, int64_t t) {
  const int64_t e = position_of(p, t);
  const int64_t row = p.rows ? (int64_t)p.rows[t] : t / p.tokens_per_row;
  if (e < 0 || e >= p.entries || row < 0 || row >= p.table_rows) return -1;
  const int col = divide((int)e, p.page);
  const int32_t page = p.tables[row * p.table_stride + col];
  if (page < 0 || page >= p.cache.pages) return -1;
  const int64_t at = page * p.cache.stride_page + ((int)e - col * p.page.d) * p.cache.stride_slot;
  return p.cache.dtype == TF_CACHE_BF16 ? at * 2 : at;
}

__device__ __forceinline__ float as_f32(float x) { return x; }
__device__ __forceinline__ float as_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* to, float x) { *to = x; }
__device__ __forceinline__ void put(__nv_bfloat16* to, float x) { *to = __float2bfloat16_rn(x); }

// One element or pair per thread: any head size and alignment.
template <typename T>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const RotaryArgs p) {
  griddep_wait();
  griddep_launch_dependents();
  const int half = p.rot / 2, items = half + (p.d - p.rot);
  const int64_t total = p.tokens * p.heads * items;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / items, t = row / p.heads;
    const int item = (int)(i - row * items), head = (int)(row - t * p.heads);
    const T* src = reinterpret_cast<const T*>(p.q) + t * p.q_ldt + head * p.q_ldh;
    T* dst = reinterpret_cast<T*>(p.q_out) + t * p.qo_ldt + head * p.qo_ldh;
    if (item < half) {
      const int i0 = p.interleaved ? 2 * item : item, i1 = p.interleaved ? 2 * item + 1 : item + half;
      const float a = as_f32(src[i0]), b = as_f32(src[i1]);
      const float2 cs = cos_sin(p, position_of(p, t), item);
      put(dst + i0, fmaf(a, cs.x, -(b * cs.y)));
      put(dst + i1, fmaf(b, cs.x, a * cs.y));
    } else {
      const int e = p.rot + item - half;
      dst[e] = src[e];  // a copy keeps its bits
    }
  }
}

// ---- whole vectors -----------------------------------------------------------------------------------------------------------------
// A block takes rows (token, head) in the tensor's order, `lanes` threads a row and 16 elements a thread, as vectors of 16 bytes that lie
// `step` elements apart, so that neighbouring threads' vectors are neighbours. Cosines and sines of the block's tokens are computed once, into
// shared memory, while the rows' loads are in flight; their order there puts neighbouring threads into different banks (in the order of the pairs
// 8192 x 64 x 128 bf16 took 54 us, now 41: the copy rate). HBM-bound.

template <typename T>
struct Vectors {
  static constexpr int kElems = 16 / (int)sizeof(T), kCount = 16 / kElems;  // of a vector; vectors
  uint4 w[kCount];
  __device__ __forceinline__ float get(int v, int e) const {
    const uint32_t* y = reinterpret_cast<const uint32_t*>(&w[v]);
    if constexpr (sizeof(T) == 4) return __uint_as_float(y[e]);
    return e & 1 ? bf16hi_to_f32(y[e >> 1]) : bf16lo_to_f32(y[e >> 1]);
  }
  // elements e and e + 1
  __device__ __forceinline__ void set2(int v, int e, float a, float b) {
    uint32_t* y = reinterpret_cast<uint32_t*>(&w[v]);
    if constexpr (sizeof(T) == 4)
      y[e] = __float_as_uint(a), y[e + 1] = __float_as_uint(b);
    else
      y[e >> 1] = pack_bf16x2(a, b);
  }
};

struct VectorPlan {
  int lanes_log2;      // threads of a row: the power of two that holds its vectors
  int items;           // threads that have 16 elements of it
  Divisor heads, half; // rows of a token; pairs of a head
  int max_tokens;      // that one block's rows touch
  int staged;          // where in shared memory the block's rows are
  int lanes, table;    // cosines of pair i of a token: at (i % p) * lanes + i / p of its `table` ones, p pairs in a vector
};

// How a thread comes by the other half of its pairs: it has them (half layout, halves of whole vectors; interleaved), or reads them from the row in shared
// memory (half layout, any rot).
enum { kHalves, kNeighbours, kStaged };

template <typename T, bool kAppend, int kMode, int kRows, int kBlocks>
__global__ void __launch_bounds__(kRotaryThreads, kBlocks) rotary_vector_kernel(const RotaryArgs p, const VectorPlan plan) {
  using X = Vectors<T>;
  constexpr bool kInterleaved = kMode == kNeighbours;
  constexpr int kE = X::kElems, kV = X::kCount, kPairs = kInterleaved ? kE / 2 : kE;
  extern __shared__ __align__(16) uint8_t smem[];
  float2* table = reinterpret_cast<float2*>(smem);
  int64_t* entry = reinterpret_cast<int64_t*>(table + plan.max_tokens * plan.table);  // [tokens of the block] where keys and values go
  [[maybe_unused]] T* staged = reinterpret_cast<T*>(smem + plan.staged);               // [rows of the block][d]
  griddep_wait();
  griddep_launch_dependents();  // what follows (attention over the cache) may take its place while this call's few blocks run
  const int slots = kRotaryThreads >> plan.lanes_log2, slot = threadIdx.x >> plan.lanes_log2, item = threadIdx.x & ((1 << plan.lanes_log2) - 1);
  const int64_t r0 = (int64_t)blockIdx.x * (slots * kRows), t0 = r0 / p.heads;
  const int first = (int)(r0 - t0 * p.heads), half = p.rot / 2;
  int tokens = divide(first + slots * kRows - 1, plan.heads) + 1;
  if (tokens > p.tokens - t0) tokens = (int)(p.tokens - t0);
  if constexpr (kAppend)  // the longest chain of loads (position, page) goes first, in the warp that
    // has the fewest angles to make (64 tokens of 80 heads 3.1 -> 2.75 us, 8000 of 48 into e4m3 24.4 -> 23.9)
    for (int t = kRotaryThreads - 1 - (int)threadIdx.x; t < tokens; t += kRotaryThreads) entry[t] = entry_offset(p, t0 + t);

  // this thread's vectors of a row lie at base + v * step. Half layout: vectors v and v + kV / 2 are pairs' two halves, or, from rot on, copied
  const bool pairs = kMode != kHalves || item * 16 < p.rot;
  const int base = pairs ? item * kE : p.rot + (item - p.rot / 16) * kE, step = kMode != kHalves ? p.d / kV : pairs ? p.rot / kV : (p.d - p.rot) / kV;
  X x[kRows];
  int token[kRows], head[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int r = first + slot + u * slots;
    token[u] = divide(r, plan.heads);
    head[u] = r - token[u] * p.heads;
    const int64_t t = t0 + token[u];
    if (item >= plan.items || t >= p.tokens) {
      token[u] = -1;
      continue;
    }
    const T* src = reinterpret_cast<const T*>(p.q) + t * p.q_ldt + head[u] * p.q_ldh;
    if constexpr (kAppend) {
      const int h = head[u] - p.q_heads, kv = (int)p.cache.kv_heads;
      if (h >= 0) src = reinterpret_cast<const T*>(h < kv ? p.k + t * p.k_ldt + h * p.k_ldh : p.v + t * p.v_ldt + (h - kv) * p.v_ldh);
    }
#pragma unroll
    for (int v = 0; v < kV; ++v) {
      x[u].w[v] = *reinterpret_cast<const uint4*>(src + base + v * step);
      if constexpr (kMode == kStaged) *reinterpret_cast<uint4*>(staged + (slot + u * slots) * p.d + base + v * step) = x[u].w[v];
    }
  }
  for (int i = threadIdx.x; i < tokens * half; i += kRotaryThreads) {
    const int t = divide(i, plan.half), pair = i - t * half;
    table[t * plan.table + (pair & (kPairs - 1)) * plan.lanes + pair / kPairs] = cos_sin(p, position_of(p, t0 + t), pair);
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    if (token[u] < 0) continue;
    const int64_t t = t0 + token[u];
    const int kv = kAppend ? (int)p.cache.kv_heads : 0, h = head[u] - p.q_heads;
    const bool turn = pairs && (!kAppend || h < kv);
    const float2* cs = table + token[u] * plan.table;
    // `put(v, e, a, b)` receives elements e and e + 1 of vector v, turned
    auto turned = [&](auto put) {
      const X y = x[u];
      [[maybe_unused]] auto neighbours = [&](int v, int e, float2 c0) {
        const float a = y.get(v, e), b = y.get(v, e + 1);
        put(v, e, fmaf(a, c0.x, -(b * c0.y)), fmaf(b, c0.x, a * c0.y));
      };
#pragma unroll
      for (int v = 0; v < (kMode != kHalves ? kV : kV / 2); ++v) {
        const float2* c = cs + (base + v * step) / kE;
        [[maybe_unused]] const int left = p.rot - (base + v * step);
        if constexpr (kInterleaved) {  // what a vector has beyond rot is copied: it keeps its bits
          if (left <= 0) continue;
          if (left >= kE) {
#pragma unroll
            for (int e = 0; e < kE; e += 2) neighbours(v, e, c[e / 2 * plan.lanes]);
            continue;
          }
        }
#pragma unroll
        for (int e = 0; e < kE; e += 2) {
          if constexpr (kMode == kStaged) {
            const T* row = staged + (slot + u * slots) * p.d;
            float z[2] = {y.get(v, e), y.get(v, e + 1)};
            const int j0 = base + v * step + e;
            if (j0 >= p.rot) continue;  // copied: keeps its bits (rot is even)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int j = j0 + i, pair = j < half ? j : j - half;
              const float2 c0 = cs[(pair & (kPairs - 1)) * plan.lanes + pair / kPairs];
              z[i] = j < half ? fmaf(z[i], c0.x, -(as_f32(row[j + half]) * c0.y)) : fmaf(z[i], c0.x, as_f32(row[j - half]) * c0.y);
            }
            put(v, e, z[0], z[1]);
          } else if constexpr (kInterleaved) {
            if (e < left) neighbours(v, e, c[e / 2 * plan.lanes]);
          } else {
            const float2 c0 = c[e * plan.lanes], c1 = c[(e + 1) * plan.lanes];
            const float a0 = y.get(v, e), b0 = y.get(v + kV / 2, e), a1 = y.get(v, e + 1), b1 = y.get(v + kV / 2, e + 1);
            put(v, e, fmaf(a0, c0.x, -(b0 * c0.y)), fmaf(a1, c1.x, -(b1 * c1.y)));
            put(v + kV / 2, e, fmaf(b0, c0.x, a0 * c0.y), fmaf(b1, c1.x, a1 * c1.y));
          }
        }
      }
    };
    T* dst = reinterpret_cast<T*>(p.q_out) + t * p.qo_ldt + head[u] * p.qo_ldh;
    if (kAppend && h >= 0) {
      const int64_t at = entry[token[u]];
      if (at < 0) continue;
      const int hh = h < kv ? h : h - kv;
      uint8_t* to = static_cast<uint8_t*>(h < kv ? p.cache.k : p.cache.v) + at;
      if (p.cache.dtype == TF_CACHE_E4M3) {
        const float* scales = h < kv ? p.cache.k_scale : p.cache.v_scale;
        const float s = scales ? __frcp_rn(load_f32(scales + hh)) : 1.0f;
        float y[kV][kE];
#pragma unroll
        for (int v = 0; v < kV; ++v)
#pragma unroll
          for (int e = 0; e < kE; ++e) y[v][e] = x[u].get(v, e);
        if (turn) turned([&](int v, int e, float a, float b) { y[v][e] = a, y[v][e + 1] = b; });
#pragma unroll
        for (int v = 0; v < kV; ++v) {
          uint32_t codes[kE / 4];
#pragma unroll
          for (int e = 0; e < kE; e += 4) codes[e / 4] = cvt_e4m3x4(y[v][e] * s, y[v][e + 1] * s, y[v][e + 2] * s, y[v][e + 3] * s);
          if constexpr (kE == 8) *reinterpret_cast<uint2*>(to + hh * p.cache.stride_head + base + v * step) = make_uint2(codes[0], codes[1]);
        }
        continue;
      }
      dst = reinterpret_cast<T*>(to) + hh * p.cache.stride_head;
    } else if (!pairs && p.in_place) {
      continue;
    }
    if (turn) turned([&](int v, int e, float a, float b) { x[u].set2(v, e, a, b); });
#pragma unroll
    for (int v = 0; v < kV; ++v) *reinterpret_cast<uint4*>(dst + base + v * step) = x[u].w[v];
  }
}

// Dependents where one block an SM is enough: 16 sequences of 1000 in a decoder layer 56.2 -> 52.4 us, 64 of 2000 167.4 -> 165.9 (captured; the attention behind
// them starts early too).
template <typename T, bool kAppend, int kRows, int kBlocks>
static tf_status launch_rotary_rows(const RotaryArgs& p, VectorPlan plan, cudaStream_t stream) {
  plan.heads = divisor(p.heads);
  plan.half = divisor(p.rot > 0 ? p.rot / 2 : 1);
  const int rows = (kRotaryThreads >> plan.lanes_log2) * kRows;
  plan.max_tokens = (rows + p.heads - 2) / p.heads + 1;
  const int64_t blocks = (p.tokens * p.heads + rows - 1) / rows;
  if (blocks > INT32_MAX) return fail(TF_ERR_UNSUPPORTED, "%s: %lld rows are too many", __func__, (long long)(p.tokens * p.heads));
  const int per = Vectors<T>::kElems / (p.interleaved ? 2 : 1);
  plan.lanes = (p.rot / 2 + per - 1) / per;
  plan.table = per * plan.lanes;
  size_t smem = (size_t)plan.max_tokens * (plan.table * sizeof(float2) + (kAppend ? sizeof(int64_t) : 0));
  auto kernel = p.interleaved ? rotary_vector_kernel<T, kAppend, kNeighbours, kRows, kBlocks> : rotary_vector_kernel<T, kAppend, kHalves, kRows, kBlocks>;
  if constexpr (kRows == 1) {
    if (!p.interleaved && p.rot % 16) {  // at most 16 KB of angles, 4 of entries and 16 of rows
      plan.staged = (int)((smem + 15) / 16 * 16);
      smem = plan.staged + (size_t)rows * p.d * sizeof(T);
      kernel = rotary_vector_kernel<T, kAppend, kStaged, kRows, kBlocks>;
    }
  }
  TF_CUDA(launch_dependent(blocks <= sm_count(), kernel, dim3((unsigned)blocks), dim3(kRotaryThreads), smem, stream, p, plan));
  return TF_OK;
}

// Two rows a thread keep the loads of a long call in flight (8192 x 64 x 128 bf16: 40.8 us with five blocks an SM, 43.2 with four; one row 42.3 to 54;
// 1777 x 20 x 80 f32 5.2 us, one row 5.8); a call that two rows would not spread over two blocks an SM takes one (4 tokens of 10 heads 2.1 -> 2.0 us;
// 64 of 80 into a cache 2.75 and 2.85: either will do). The append kernel spills at five blocks and the f32 one is slower (by a quarter).
template <typename T, bool kAppend>
static tf_status launch_rotary_vectors(const RotaryArgs& p, cudaStream_t stream) {
  VectorPlan plan = {};
  plan.items = p.d / 16;
  while ((1 << plan.lanes_log2) < plan.items) ++plan.lanes_log2;
  const int64_t two = (int64_t)(kRotaryThreads >> plan.lanes_log2) * 2;
  if (p.tokens * p.heads <= two * 2 * sm_count() || (!p.interleaved && p.rot % 16)) return launch_rotary_rows<T, kAppend, 1, sizeof(T) == 2 ? 6 : 4>(p, plan, stream);
  return launch_rotary_rows<T, kAppend, 2, !kAppend && sizeof(T) == 2 ? 5 : kAppend ? 3 : 4>(p, plan, stream);
}

template <typename T>
static tf_status launch_rotary(const RotaryArgs& p, cudaStream_t stream) {
  // Whole vectors need 16-byte aligned rows of whole vectors.
  const int64_t unit = 16 / (int64_t)sizeof(T);
  auto aligned = [&](const void* x, int64_t a, int64_t b) { return reinterpret_cast<uintptr_t>(x) % 16 == 0 && a % unit == 0 && b % unit == 0; };
  if (p.d % 16 == 0 && aligned(p.q, p.q_ldt, p.q_ldh) && aligned(p.q_out, p.qo_ldt, p.qo_ldh)) return launch_rotary_vectors<T, false>(p, stream);
  const int64_t total = p.tokens * p.heads * (p.d - p.rot / 2), cap = (int64_t)sm_count() * 8;
  const int64_t need = (total + kRotaryThreads - 1) / kRotaryThreads;
  TF_CUDA(launch_dependent(need <= sm_count(), rotary_kernel<T>, dim3((unsigned)(need < cap ? need : cap)), dim3(kRotaryThreads), 0, stream, p));
  return TF_OK;
}

}  // namespace tf
