// Attention of new tokens over a paged key-value cache, split over its length and joined.
//
// The rows of one kv head (its query heads times the new tokens) read the same keys, so keys stream through once, as the 16-row operand of
// mma.sync m16n8k16: S^T = K Q^T and O^T = V^T P^T, rows in eights. (Rows as the 16-row operand took twice the products and accumulators for the
// eight rows that most models have.) Bound by HBM: a bf16 key and value of 128 elements are 512 bytes for 512 operations per row, while the products of
// eight rows keep the tensor pipe 15 % busy.
//
// One pass with a running maximum and sum (base 2, f32). The workers are single warps, or teams of 2 or 4 warps with rows of their own where
// one warp's registers do not hold them. Each has a ring of its own in shared memory, filled by cp.async, and never waits for another: while one waits for a
// head's first keys, the others of its SM keep the memory busy.
//
// The work is the list of all (sequence, row tile, kv head), each as long as its tiles of keys and a fixed part for starting it, cut into as many
// equal contiguous ranges as there are workers, whatever the lengths are (they are read on the device, so a captured call follows them). A worker
// that has seen all keys of a head writes its result. Else it leaves its maximum, sum and unnormalised sum of values in the workspace (one for all
// workers of a block that lies inside a head), and paged_attention_join_kernel adds them up in the order of the keys.
//
// Measured (CUDA graph, device time): 64 sequences of up to 8192 entries, 8 kv heads of 128, eight query heads each: bf16 178 us = 6.4 TB/s of keys and values,
// 0.98 of a copy's rate; two of 131072 109 us, 0.98; e4m3, 32 of up to 16384, 97 us, 0.93 (with 16-bit operands to make); 40 rows of 96 elements 42 us
// against 16 of HBM time, bound by products and softmax of two warps a scheduler taking turns; calls of a few microseconds by their chain of
// loads (lengths, page, keys; parts) and two launches: one sequence of 129 entries 7.6 us.
#pragma once

#include <cmath>
#include <type_traits>

#include "paged_attention.h"

namespace tf {

constexpr int kAttendWarps = 4, kAttendThreads = 32 * kAttendWarps;
constexpr int kHeadCost = 4;  // what starting a head costs a worker, in tiles: 3 to 5 us to its first keys, a tile 1 to 2 (192 short sequences 30.2 us with 2, 26.4 with 4)

// ROWS query rows of a kv head, in eights: as many of them to a warp as its registers hold (an accumulator of DP x 8 takes DP / 4 of them), the rest to
// a team of warps that share the keys' tiles.
template <int DP, bool F8, int ROWS>
struct AttendCfg {
  static constexpr int kEights = DP == 256 ? (ROWS > 8 ? 2 : 1) : ROWS <= 32 ? ROWS / 8 : ROWS / 16, kTeam = ROWS / (8 * kEights);
  static constexpr int kTeams = kAttendWarps / kTeam, kRows = ROWS;
  static constexpr int kItem = F8 ? 1 : 2, kRowBytes = (DP <= 64 ? 64 : DP <= 128 ? 128 : 256) * kItem;  // of a staged row: a power of two
  // The query operand takes half the accumulators' registers. Where both do not fit it is read from shared memory with every tile.
  static constexpr bool kQueriesInRegisters = kEights * DP <= 384;
  static constexpr int kQueryBytes = kQueriesInRegisters ? 0 : 8 * kEights * (DP <= 64 ? 64 : DP <= 128 ? 128 : 256) * 2;  // of a warp
  // Keys of a team's tile: a tile costs as much as the products of eight rows do besides its keys, so 32 where two stages of them fit (12 sequences of up to 16384:
  // e4m3 8 rows of 128 elements 39 -> 35 us, 16 40 -> 37, 24 49 -> 44; bf16 48 rows of 96 76 -> 67).
  static constexpr int kKeys = kRowBytes <= 128 || (kTeam == 2 && kRowBytes <= 256) ? 32 : 16;
  static constexpr int kLoadRows = kKeys / kTeam;  // of them, a warp loads
  static constexpr int kHalf = kKeys * kRowBytes;  // the keys of a tile, or its values
  // three blocks an SM where the registers allow it without spilling (64 x 8192 bf16 183 us, 187 with two and a third stage)
  static constexpr int kBlocksPerSm = DP == 256 && !F8 ? 1 : kEights * DP <= 128 ? 3 : 2;
  static constexpr int kFit = (200704 - kBlocksPerSm * kAttendWarps * kQueryBytes) / (kBlocksPerSm * kTeams * 2 * kHalf);
  static constexpr int kStages = kFit < 2 ? 2 : kFit > 6 ? 6 : kFit;
  static constexpr int kRing = kTeams * kStages * 2 * kHalf, kParts = kTeams * kRows * (DP + 2) * 4;  // kParts: what a block joins of its own
  static constexpr int kSmem = kRing + kAttendWarps * kQueryBytes > kParts ? kRing + kAttendWarps * kQueryBytes : kParts;
  static constexpr int kChunks = kRowBytes / 16;      // of a staged row
  static constexpr int kRowsPerCopy = 32 / kChunks;   // rows that one copy instruction of a warp covers
  static_assert(kBlocksPerSm * (kSmem + 2560) <= 228 * 1024 && kSmem <= 225 * 1024, "the grid counts on so many blocks an SM");
  // An e4m3 entry is multiplied as f16: weights are scaled by 2^kShift, so that the largest is above 2^6 and at most 2^15, and small ones keep their bits.
  static constexpr float kSlack = 8.0f;
  static constexpr float kShift = F8 ? 15.0f - kSlack : 0.0f;
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 16 bytes global -> shared without registers, where `on`; zeros where `bytes` is 0 (the address is then not read).
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, int bytes, bool on) {
  asm volatile("{ .reg .pred p;\n setp.ne.s32 p, %3, 0;\n @p cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2; }" ::"r"(dst), "l"(src), "r"(bytes), "r"((int)on) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void load_matrices_turned(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <bool F16>
__device__ __forceinline__ void multiply(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// an 8 x 8 matrix of 16-bit elements, two neighbours of a row per thread, turned
__device__ __forceinline__ uint32_t turn_matrix(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// two e4m3 codes (the lower or upper half of a word) -> two f16, exactly
__device__ __forceinline__ uint32_t codes_to_f16x2(uint32_t w, bool upper) {
  uint32_t r;
  if (upper)
    asm("{ .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %1;\n cvt.rn.f16x2.e4m3x2 %0, hi; }" : "=r"(r) : "r"(w));
  else
    asm("{ .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %1;\n cvt.rn.f16x2.e4m3x2 %0, lo; }" : "=r"(r) : "r"(w));
  return r;
}
template <int TEAM>
__device__ __forceinline__ void team_sync(int team) {
  if constexpr (TEAM == 1)
    __syncwarp();
  else
    asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(32 * TEAM) : "memory");
}

// What the rows of one row tile of one sequence see: keys [lo, hi) between them. The first row's limit is `first`, the last real row's hi.
struct Span {
  int start, hi, units;  // start: lo rounded down to a whole unit
  int first, last_lo;    // every row sees [last_lo, first)
  int length, count;
};

template <int ROWS, int UNIT>
__device__ __forceinline__ Span span_of(const AttendArgs& p, int index) {
  const int b = p.row_tiles == 1 ? index : index / p.row_tiles, tile = p.row_tiles == 1 ? 0 : index - b * p.row_tiles;
  Span s;
  const int len = p.lengths[b], cnt = p.counts ? p.counts[b] : p.queries;
  s.length = len < 0 ? 0 : len > p.entries ? p.entries : len;
  s.count = cnt < 0 ? 0 : cnt > p.queries ? p.queries : cnt;
  int i0 = 0, i1 = s.count - 1;  // the tile's first and last real query
  if (p.row_tiles > 1) {
    const int r0 = tile * ROWS;
    int r1 = p.queries * p.group.d - 1;
    if (r1 > r0 + ROWS - 1) r1 = r0 + ROWS - 1;
    i0 = divide(r0, p.group);
    if (i1 > divide(r1, p.group)) i1 = divide(r1, p.group);
  }
  s.start = s.hi = s.units = s.first = s.last_lo = 0;
  if (i0 > i1) return s;
  const int base = s.length - s.count + 1;
  s.first = base + i0;
  s.hi = base + i1;
  if (s.hi <= 0) {
    s.hi = 0;
    return s;
  }
  int lo = 0;
  if (p.window > 0) {
    lo = s.first > p.window ? s.first - p.window : 0;
    s.last_lo = s.hi > p.window ? s.hi - p.window : 0;
  }
  s.start = lo / UNIT * UNIT;
  s.units = (s.hi - s.start + UNIT - 1) / UNIT;
  return s;
}

// n / d, with the short division where both fit it.
__device__ __forceinline__ long long quotient(long long n, long long d) {
  return ((n | d) >> 32) == 0 ? (long long)((uint32_t)n / (uint32_t)d) : n / d;
}

// `total` positions dealt out to workers in contiguous ranges that differ by one at most; none of them is empty.
struct Ranges {
  long long each, more;  // the first `more` workers have each + 1
  int workers;
  __device__ static Ranges of(long long total, int most) {
    Ranges r;
    r.workers = total < most ? (int)total : most;
    r.each = r.workers ? quotient(total, r.workers) : 0;
    r.more = total - r.each * r.workers;
    return r;
  }
  __device__ long long begin(int w) const { return each * w + (w < more ? w : more); }
  __device__ int of_position(long long x) const {
    const long long large = (each + 1) * more;
    return (int)(x < large ? quotient(x, each + 1) : more + quotient(x - large, each));
  }
};

// Writes the results of eight rows, from `row` on, whose sums are in the registers' order: a thread has rows 2c and 2c + 1, c = lane % 4, of elements
// 16 t + lane / 4 and 8 more, or, of e4m3 values, 16 t + 2 (lane / 4) and one more.
template <bool F8>
struct Finish {
  float scale[2];
  bool nothing[2];
  __nv_bfloat16* out;  // of row lane / 4
  int64_t lse[2];      // -1: there is no such row
  bool real;
  __device__ __forceinline__ Finish(const AttendArgs& p, const Span& sp, int b, int kv, int row, float v_scale, float2 sum) {
    const int lane = threadIdx.x & 31, rows = p.queries * p.group.d;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = row + 2 * (lane & 3) + h, i = divide(r, p.group);
      const float l = h ? sum.y : sum.x;
      nothing[h] = l == 0.0f || i >= sp.count;  // padding goes along unmasked
      scale[h] = v_scale / l;
      lse[h] = r < rows ? ((int64_t)b * p.queries + i) * p.q_heads + kv * p.group.d + r - i * p.group.d : -1;
    }
    const int r = row + (lane >> 2), i = divide(r, p.group);
    real = r < rows;
    out = p.out + ((int64_t)b * p.queries + i) * p.out_ldt + ((int64_t)kv * p.group.d + r - i * p.group.d) * p.out_ldh;
  }
  __device__ __forceinline__ void write_lse(const AttendArgs& p, float2 top, float2 sum, float shift) const {
    if (!p.lse) return;
    if (lse[0] >= 0) p.lse[lse[0]] = nothing[0] ? -INFINITY : (top.x + log2f(sum.x) - shift) * 0.6931471805599453f;
    if (lse[1] >= 0) p.lse[lse[1]] = nothing[1] ? -INFINITY : (top.y + log2f(sum.y) - shift) * 0.6931471805599453f;
  }
  __device__ __forceinline__ void write(const AttendArgs& p, int t, float4 x) const {
    const int c = threadIdx.x & 3;
    const uint32_t w0 = turn_matrix(pack_bf16x2(nothing[0] ? 0.0f : x.x * scale[0], nothing[1] ? 0.0f : x.y * scale[1]));
    const uint32_t w1 = turn_matrix(pack_bf16x2(nothing[0] ? 0.0f : x.z * scale[0], nothing[1] ? 0.0f : x.w * scale[1]));
    if (!real || 16 * t >= p.d) return;
    if constexpr (F8) {  // even and odd elements 4c, 4c + 2 and 4c + 1, 4c + 3
      *reinterpret_cast<uint2*>(out + 16 * t + 4 * c) = make_uint2(__byte_perm(w0, w1, 0x5410), __byte_perm(w0, w1, 0x7632));
    } else {
      *reinterpret_cast<uint32_t*>(out + 16 * t + 2 * c) = w0;
      *reinterpret_cast<uint32_t*>(out + 16 * t + 8 + 2 * c) = w1;
    }
  }
};

template <int DP, bool F8, int ROWS>
__global__ void __launch_bounds__(kAttendThreads, (AttendCfg<DP, F8, ROWS>::kBlocksPerSm)) paged_attention_kernel(const AttendArgs p) {
  using C = AttendCfg<DP, F8, ROWS>;
  constexpr int TEAM = C::kTeam, NR = C::kEights, KT = C::kKeys / 16;
  constexpr bool kInRegisters = C::kQueriesInRegisters;
  extern __shared__ __align__(1024) uint8_t smem[];  // rows of the ring start on multiples of their size
  __shared__ uint32_t s_seen[C::kTeams][C::kStages][TEAM];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, team = warp / TEAM, member = warp % TEAM;
  griddep_wait();
  griddep_launch_dependents();  // the join: its blocks find room as this kernel's leave
  const int worker = blockIdx.x * C::kTeams + team;

  // The workers' ranges of the list, and where in it this one's begins: every lane takes a few neighbouring spans, every warp for itself.
  auto cost_of = [&](int i) {
    const int units = i < p.spans ? span_of<C::kRows, C::kKeys>(p, i).units : 0;
    return units ? units + kHeadCost : 0;
  };
  const int share = (p.spans + 31) / 32;
  long long cost = cost_of(lane * share);
#pragma unroll 8
  for (int i = 1; i < share; ++i) cost += cost_of(lane * share + i);
  long long upto = cost;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    const long long y = __shfl_up_sync(~0u, upto, x);
    if (lane >= x) upto += y;
  }
  const Ranges ranges = Ranges::of(__shfl_sync(~0u, upto, 31) * p.kv_heads, (int)gridDim.x * C::kTeams);
  if (worker >= ranges.workers) return;
  const long long u0 = ranges.begin(worker), u1 = ranges.begin(worker + 1);
  const int owner = __popc(__ballot_sync(~0u, upto * p.kv_heads <= u0));  // the lane whose spans u0 falls into
  int index = owner * share;
  long long before = __shfl_sync(~0u, upto - cost, owner) * p.kv_heads;  // where span `index` begins
  for (int at = 0; at < share && share > 1; at += 32) {  // which of them: 32 at a time
    const long long c = at + lane < share ? (long long)cost_of(owner * share + at + lane) * p.kv_heads : 0;
    long long here = c;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      const long long y = __shfl_up_sync(~0u, here, x);
      if (lane >= x) here += y;
    }
    const int passed = __popc(__ballot_sync(~0u, before + here <= u0));  // all spans that end at or before this range
    if (passed < 32) {
      index = owner * share + at + passed;
      before += __shfl_sync(~0u, here - c, passed);
      break;
    }
    before += __shfl_sync(~0u, here, 31);
  }

  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + team * C::kStages * 2 * C::kHalf;
  [[maybe_unused]] uint8_t* queries = smem + C::kRing + warp * C::kQueryBytes;  // this warp's, written and read by the same threads
  const int chunks = p.d * C::kItem / 16;  // of a staged row, that hold data
  const int copy_row = lane / C::kChunks, copy_chunk = lane % C::kChunks;
  // Chunk c of row r lies at c ^ swizzle(r): the eight rows of a matrix load are in other banks. Rows start on multiples of their size, so a
  // step to another chunk, and to a row of the same instruction's series, is an exclusive or with a constant.
  auto swizzle = [](int row) { return C::kRowBytes >= 128 ? row & 7 : (row >> 1) & 3; };
  const uint32_t copy_to = (member * C::kLoadRows + copy_row) * C::kRowBytes + ((copy_chunk ^ swizzle(member * C::kLoadRows + copy_row)) << 4);
  // matrix loads of four 8 x 8 blocks: K by (keys, keys + 8) x (chunk, chunk + 1), V in the same order for codes, turned and chunks first for bf16
  const int k_row = (lane & 7) + (lane & 8), v_row = F8 ? k_row : (lane & 7) + ((lane >> 4) << 3);
  const uint32_t k_from = k_row * C::kRowBytes + (((lane >> 4) ^ swizzle(k_row)) << 4);
  const uint32_t v_from = v_row * C::kRowBytes + (((F8 ? lane >> 4 : (lane >> 3) & 1) ^ swizzle(v_row)) << 4);

  if (p.d < DP) {
    // the products run over DP elements: the keys' others are zero, as the queries' are (the values' give columns that nobody reads)
    for (int i = lane; i < C::kStages * C::kKeys / TEAM * C::kChunks; i += 32) {
      const int ch = i % C::kChunks, r = i / C::kChunks * TEAM + member, row = r % C::kKeys;
      if (ch >= chunks)
        *reinterpret_cast<uint4*>(smem + team * C::kStages * 2 * C::kHalf + r / C::kKeys * 2 * C::kHalf + row * C::kRowBytes + ((ch ^ swizzle(row)) << 4)) =
            make_uint4(0u, 0u, 0u, 0u);
    }
  }

  for (long long u = u0; u < u1;) {
    const Span sp = span_of<C::kRows, C::kKeys>(p, index);
    if (sp.units == 0) {
      ++index;
      continue;
    }
    const int cost = sp.units + kHeadCost, kv = (int)quotient(u - before, cost), from = (int)((u - before) - (long long)kv * cost);
    const int to = cost - from < u1 - u ? cost : from + (int)(u1 - u);
    const int unit = from > kHeadCost ? from - kHeadCost : 0, tiles = to - kHeadCost - unit;
    const int span = index;
    const int64_t slot = 2 * (int64_t)worker + (u == u0 ? 0 : 1);
    const long long head_end = before + (long long)(kv + 1) * cost;
    u += to - from;
    if (u == before + (long long)cost * p.kv_heads) {
      before = u;
      ++index;
    }
    if (tiles <= 0) continue;
    if (unit == 0 && lane == 0 && member == 0) p.shares[(int64_t)span * p.kv_heads + kv] = make_int4(worker, ranges.of_position(head_end - 1), (int)slot, 0);
    const int b = p.row_tiles == 1 ? span : span / p.row_tiles, row0 = (span - b * p.row_tiles) * C::kRows;
    const int key0 = sp.start + unit * C::kKeys;

    // The lanes hold 64 neighbouring entries of the table, asked for long before they are used.
    const int32_t* table = p.tables + b * p.table_stride;
    const int last_column = divide(sp.hi - 1, p.page);
    auto entries_at = [&](int column) { return column + lane <= last_column ? table[column + lane] : -1; };
    int column0 = divide(key0, p.page), entries0 = entries_at(column0), entries1 = entries_at(column0 + 32);
    const uint8_t* kbase = p.k + kv * p.stride_head + copy_chunk * 16;
    const uint8_t* vbase = p.v + kv * p.stride_head + copy_chunk * 16;
    int fill = 0, stage = 0;  // the ring's places that are filled and read next
    auto issue = [&](int tile) {
      if (tile < tiles) {
        const int first = key0 + tile * C::kKeys, column = divide(first, p.page);
        if (column - column0 >= 32) {  // a tile has at most 32 pages
          column0 += 32;
          entries0 = entries1;
          entries1 = entries_at(column0 + 32);
        }
        const uint32_t to = ring + fill * 2 * C::kHalf + copy_to;
        uint32_t seen;
        if (p.whole_tiles) {  // pages hold whole tiles: one page for all rows
          const int page = __shfl_sync(~0u, entries0, column - column0), many = sp.hi - first < C::kKeys ? sp.hi - first : C::kKeys;
          const bool ok = page >= 0 && page < p.pages;
          seen = ok ? (uint32_t)((1ull << many) - 1) : 0u;
          int64_t o = ok ? page * p.stride_page + (int64_t)(first - column * p.page.d + member * C::kLoadRows + copy_row) * p.stride_slot : 0;
          const int left = ok ? many - member * C::kLoadRows - copy_row : 0;
#pragma unroll
          for (int i = 0; i < (C::kLoadRows + C::kRowsPerCopy - 1) / C::kRowsPerCopy; ++i) {
            const bool on = copy_chunk < chunks && (C::kLoadRows % C::kRowsPerCopy == 0 || i * C::kRowsPerCopy + copy_row < C::kLoadRows);
            const uint32_t dst = (to ^ (swizzle(i * C::kRowsPerCopy) << 4)) + i * C::kRowsPerCopy * C::kRowBytes;
            const bool have = i * C::kRowsPerCopy < left;
            const int64_t at = have ? o : 0;
            copy_async(dst, kbase + at, have ? 16 : 0, on);
            copy_async(dst + C::kHalf, vbase + at, have ? 16 : 0, on);
            o += (int64_t)C::kRowsPerCopy * p.stride_slot;
          }
        } else {
          const int key = first + member * C::kLoadRows + lane, col = divide(key, p.page), at = col - column0;
          const int e0 = __shfl_sync(~0u, entries0, at & 31), e1 = __shfl_sync(~0u, entries1, at & 31), page = at < 32 ? e0 : e1;
          const bool ok = lane < C::kLoadRows && key < sp.hi && page >= 0 && page < p.pages;
          const int64_t off = ok ? page * p.stride_page + (int64_t)(key - col * p.page.d) * p.stride_slot : 0;
          seen = __ballot_sync(~0u, ok);
#pragma unroll
          for (int i = 0; i < (C::kLoadRows + C::kRowsPerCopy - 1) / C::kRowsPerCopy; ++i) {
            const int r = i * C::kRowsPerCopy + copy_row;  // of this warp's rows
            const int64_t o = __shfl_sync(~0u, off, r & 31);
            const int bytes = (seen >> (r & 31)) & 1 ? 16 : 0;
            const bool on = copy_chunk < chunks && (C::kLoadRows % C::kRowsPerCopy == 0 || r < C::kLoadRows);
            const uint32_t dst = (to ^ (swizzle(i * C::kRowsPerCopy) << 4)) + i * C::kRowsPerCopy * C::kRowBytes;
            copy_async(dst, kbase + o, bytes, on);
            copy_async(dst + C::kHalf, vbase + o, bytes, on);
          }
          seen <<= member * C::kLoadRows;
        }
        if (lane == 0) s_seen[team][fill][member] = seen;
        fill = fill + 1 == C::kStages ? 0 : fill + 1;
      }
      copy_commit();
    };
    // The query operand: row lane / 4 of each eight, asked for before the copies wait for the table. Scores and sums are of rows 2c and 2c + 1, c = lane % 4.
    uint32_t qf[DP / 16][NR][2];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const int r = row0 + member * 8 * NR + 8 * n + (lane >> 2), i = divide(r, p.group);
      const bool real = r < p.queries * p.group.d;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(p.q + ((int64_t)b * p.queries + i) * p.q_ldt + ((int64_t)kv * p.group.d + r - i * p.group.d) * p.q_ldh);
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        // a matrix load of e4m3 codes leaves four neighbours in a thread: elements 4c .. 4c + 3 stand at k = 2c, 2c + 1, 2c + 8, 2c + 9
        if constexpr (F8) {
          const uint2 w = real && kk * 16 < p.d ? *reinterpret_cast<const uint2*>(src + kk * 8 + (lane & 3) * 2) : make_uint2(0u, 0u);
          qf[kk][n][0] = w.x, qf[kk][n][1] = w.y;
        } else {
          qf[kk][n][0] = real && kk * 16 < p.d ? src[kk * 8 + (lane & 3)] : 0u;
          qf[kk][n][1] = real && kk * 16 < p.d ? src[kk * 8 + (lane & 3) + 4] : 0u;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < C::kStages - 1; ++i) issue(i);
    float row_scale[NR][2];
    int limit[NR][2], lowest[NR][2];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      row_scale[n][0] = row_scale[n][1] = p.scale_log2;
      if constexpr (F8) {
        // bf16 -> f16: the row is scaled by a power of two that puts its largest element into [2^14, 2^15), or by 2^126 (its scores are zero to f32 then). Elements of
        // at least 2^-31 of that one keep all their bits, those below 2^-39 become zero
        float top = 0.0f;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
          for (int x = 0; x < 2; ++x) top = fmaxf(top, fmaxf(fabsf(bf16lo_to_f32(qf[kk][n][x])), fabsf(bf16hi_to_f32(qf[kk][n][x]))));
        top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
        top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
        const int e = (int)(__float_as_uint(top) >> 23);  // biased exponent; 0 and infinities are left as they are
        int up = e == 0 || e == 255 ? 0 : 127 + 14 - e;
        if (up > 126) up = 126;
        const float grow = __uint_as_float((uint32_t)(127 + up) << 23), shrink = __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
          for (int x = 0; x < 2; ++x) qf[kk][n][x] = pack_f16x2(bf16lo_to_f32(qf[kk][n][x]) * grow, bf16hi_to_f32(qf[kk][n][x]) * grow);
        const float mine = p.scale_log2 * (p.k_scale ? load_f32(p.k_scale + kv) : 1.0f) * shrink;
#pragma unroll
        for (int h = 0; h < 2; ++h) row_scale[n][h] = __shfl_sync(~0u, mine, (2 * (lane & 3) + h) * 4);
      }
      if constexpr (!kInRegisters) {
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)  // in the order of use: a thread's two words of a step, neighbours' behind one another
          *reinterpret_cast<uint2*>(queries + ((kk * NR + n) * 32 + lane) * 8) = make_uint2(qf[kk][n][0], qf[kk][n][1]);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r2 = row0 + member * 8 * NR + 8 * n + 2 * (lane & 3) + h, i2 = divide(r2, p.group);
        limit[n][h] = r2 < p.queries * p.group.d && i2 < sp.count ? sp.length - sp.count + 1 + i2 : 0;
        lowest[n][h] = p.window > 0 && limit[n][h] > p.window ? limit[n][h] - p.window : 0;
      }
    }
    float o[DP / 16][NR][4], m[NR][2], l[NR][2];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.0f;
#pragma unroll
      for (int t = 0; t < DP / 16; ++t) o[t][n][0] = o[t][n][1] = o[t][n][2] = o[t][n][3] = 0.0f;
    }

    for (int tile = 0; tile < tiles; ++tile) {
      copy_wait<C::kStages - 2>();
      team_sync<TEAM>(team);
      issue(tile + C::kStages - 1);
      const int key = key0 + tile * C::kKeys;
      const uint32_t kt = ring + stage * 2 * C::kHalf, vt = kt + C::kHalf;
      uint32_t seen = 0;
#pragma unroll
      for (int w = 0; w < TEAM; ++w) seen |= s_seen[team][stage][w];
      stage = stage + 1 == C::kStages ? 0 : stage + 1;

      float s[KT][NR][4];  // keys 16 j + lane / 4 (+ 8 for the upper two) of rows 2c, 2c + 1
#pragma unroll
      for (int j = 0; j < KT; ++j)
#pragma unroll
        for (int n = 0; n < NR; ++n) s[j][n][0] = s[j][n][1] = s[j][n][2] = s[j][n][3] = 0.0f;
#pragma unroll
      for (int kk = 0; kk < DP / 16; kk += F8 ? 2 : 1) {
        uint32_t q[F8 ? 2 : 1][NR][2];
#pragma unroll
        for (int y = 0; y < (F8 ? 2 : 1); ++y)
#pragma unroll
          for (int n = 0; n < NR; ++n) {
            if constexpr (kInRegisters) {
              q[y][n][0] = qf[kk + y][n][0], q[y][n][1] = qf[kk + y][n][1];
            } else {
              const uint2 w = *reinterpret_cast<const uint2*>(queries + (((kk + y) * NR + n) * 32 + lane) * 8);
              q[y][n][0] = w.x, q[y][n][1] = w.y;
            }
          }
#pragma unroll
        for (int j = 0; j < KT; ++j) {
          uint32_t r[4];
          load_matrices(r, ((kt + k_from) ^ (kk << (F8 ? 4 : 5))) + j * 16 * C::kRowBytes);
          if constexpr (F8) {
            const uint32_t a0[4] = {codes_to_f16x2(r[0], false), codes_to_f16x2(r[1], false), codes_to_f16x2(r[0], true), codes_to_f16x2(r[1], true)};
            const uint32_t a1[4] = {codes_to_f16x2(r[2], false), codes_to_f16x2(r[3], false), codes_to_f16x2(r[2], true), codes_to_f16x2(r[3], true)};
#pragma unroll
            for (int n = 0; n < NR; ++n) multiply<true>(s[j][n], a0, q[0][n][0], q[0][n][1]);
#pragma unroll
            for (int n = 0; n < NR; ++n) multiply<true>(s[j][n], a1, q[1][n][0], q[1][n][1]);
          } else {
#pragma unroll
            for (int n = 0; n < NR; ++n) multiply<false>(s[j][n], r, q[0][n][0], q[0][n][1]);
          }
        }
      }

      // Exponents relative to the row's reference. It is a maximum of earlier keys and moves only when a key passes it by 2^kSlack (or is the first that
      // is seen): weights up to that are as exact, and most tiles need neither the maximum over the warp nor the accumulators' rescaling.
      const bool whole = seen == (uint32_t)((1ull << C::kKeys) - 1);
      const bool inside = key >= sp.last_lo && key + C::kKeys <= sp.first;  // every row sees all of the tile's keys that anyone sees
      float offset[NR][2];
      bool moved = false;
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          offset[n][h] = m[n][h] == -INFINITY ? 0.0f : C::kShift - m[n][h];
#pragma unroll
          for (int j = 0; j < KT; ++j)
#pragma unroll
            for (int x = 0; x < 4; x += 2) s[j][n][x + h] = fmaf(s[j][n][x + h], row_scale[n][h], offset[n][h]);
        }
      if (!(whole && inside)) {
#pragma unroll
        for (int j = 0; j < KT; ++j)
#pragma unroll
          for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int c = 16 * j + (lane >> 2) + 8 * (x >> 1), e = key + c;
              if (!((seen >> c) & 1) || e < lowest[n][x & 1] || e >= limit[n][x & 1]) s[j][n][x] = -INFINITY;
            }
      }
      float top[NR][2];
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float t = fmaxf(s[0][n][h], s[0][n][2 + h]);
#pragma unroll
          for (int j = 1; j < KT; ++j) t = fmaxf(t, fmaxf(s[j][n][h], s[j][n][2 + h]));
          top[n][h] = t;
          moved |= t > (m[n][h] == -INFINITY ? -INFINITY : C::kShift + C::kSlack);
        }
      if (__any_sync(~0u, moved)) {
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float t = top[n][h];
            t = fmaxf(t, __shfl_xor_sync(~0u, t, 4));
            t = fmaxf(t, __shfl_xor_sync(~0u, t, 8));
            t = fmaxf(t, __shfl_xor_sync(~0u, t, 16));
            // A whole number: its differences, and the factors between parts, are exact. What was unset has offset 0.
            const float now = fmaxf(m[n][h], ceilf(t - offset[n][h]));
            const float next = now == -INFINITY ? 0.0f : C::kShift - now;
            const float keep = exp2_approx(m[n][h] - (now == -INFINITY ? 0.0f : now));
            l[n][h] *= keep;
            m[n][h] = now;
#pragma unroll
            for (int x = 0; x < DP / 16; ++x) o[x][n][h] *= keep, o[x][n][2 + h] *= keep;
#pragma unroll
            for (int j = 0; j < KT; ++j) s[j][n][h] += next - offset[n][h], s[j][n][2 + h] += next - offset[n][h];
          }
      }
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < KT; ++j) {
            s[j][n][h] = exp2_approx(s[j][n][h]), s[j][n][2 + h] = exp2_approx(s[j][n][2 + h]);
            l[n][h] += s[j][n][h] + s[j][n][2 + h];
          }

      // A value that some rows see and others do not reaches both through the product, the latter with weight 0: harmless unless it is not finite.
      bool odd = false;
      const uint8_t* values = smem + (vt - (uint32_t)__cvta_generic_to_shared(smem));
      if (!inside) {
        for (int i = lane; i < C::kKeys * chunks; i += 32) {
          const int row = i / chunks, ch = i - row * chunks;
          const uint4 w = *reinterpret_cast<const uint4*>(values + row * C::kRowBytes + ((ch ^ swizzle(row)) << 4));
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const uint32_t y = x == 0 ? w.x : x == 1 ? w.y : x == 2 ? w.z : w.w;
            if constexpr (F8)
              odd |= __vcmpeq4(y & 0x7F7F7F7Fu, 0x7F7F7F7Fu) != 0;
            else
              odd |= __vcmpgeu2(y & 0x7FFF7FFFu, 0x7F807F80u) != 0;
          }
        }
        odd = __any_sync(~0u, odd);
      }
      if (!odd) {
#pragma unroll
        for (int j = 0; j < KT; ++j) {
          uint32_t hi[NR][2];
          [[maybe_unused]] uint32_t lo[NR][2];
#pragma unroll
          for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int x = 0; x < 2; ++x) {  // scores are (key, rows); the weights' operand wants (row, keys)
              const float a = s[j][n][2 * x], c = s[j][n][2 * x + 1];
              if constexpr (F8) {
                hi[n][x] = turn_matrix(pack_f16x2(a, c));
              } else {
                // 16 bits of a weight in two products: one of 8 bits would add an error as large as the result's own rounding
                const uint32_t w = pack_bf16x2(a, c);
                hi[n][x] = turn_matrix(w);
                lo[n][x] = turn_matrix(pack_bf16x2(a - bf16lo_to_f32(w), c - bf16hi_to_f32(w)));
              }
            }
#pragma unroll
          for (int t = 0; t < DP / 16; t += F8 ? 2 : 1) {
            uint32_t r[4];
            load_matrices_turned(r, ((vt + v_from) ^ (t << (F8 ? 4 : 5))) + j * 16 * C::kRowBytes);
            if constexpr (F8) {
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                // a thread holds elements (2i, 2i + 1), i = lane / 4, of two keys: bytes to (key, key + 1) pairs; the even elements are the operand's rows i, the odd ones 8 + i
                const uint32_t w0 = __byte_perm(r[2 * x], 0, 0x3120), w1 = __byte_perm(r[2 * x + 1], 0, 0x3120);
                const uint32_t a[4] = {codes_to_f16x2(w0, false), codes_to_f16x2(w0, true), codes_to_f16x2(w1, false), codes_to_f16x2(w1, true)};
#pragma unroll
                for (int n = 0; n < NR; ++n) multiply<true>(o[t + x][n], a, hi[n][0], hi[n][1]);
              }
            } else {
#pragma unroll
              for (int n = 0; n < NR; ++n) multiply<false>(o[t][n], r, hi[n][0], hi[n][1]);
#pragma unroll
              for (int n = 0; n < NR; ++n) multiply<false>(o[t][n], r, lo[n][0], lo[n][1]);
            }
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 2 * KT; ++j)  // eight keys
#pragma unroll 1
          for (int x8 = 0; x8 < 8; ++x8) {
            const int c = 8 * j + x8;
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float w = __shfl_sync(~0u, s[j / 2][n][2 * (j & 1) + h], 4 * x8 + (lane & 3));
                if (!((seen >> c) & 1) || key + c < lowest[n][h] || key + c >= limit[n][h]) continue;
#pragma unroll
                for (int t = 0; t < DP / 16; ++t)
#pragma unroll
                  for (int x = 0; x < 2; ++x) {
                    const int e = 16 * t + (F8 ? 2 * (lane >> 2) + x : (lane >> 2) + 8 * x), byte = F8 ? e : 2 * e;
                    const uint8_t* at = values + c * C::kRowBytes + (((byte >> 4) ^ swizzle(c)) << 4) + (byte & 15);
                    const float y = F8 ? e4m3_to_f32(*at) : __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(at));
                    o[t][n][2 * x + h] = fmaf(w, y, o[t][n][2 * x + h]);
                  }
              }
          }
      }
    }

    // the result, or this worker's part of it: its registers in their order
    const bool all = tiles == sp.units;
    if constexpr (C::kTeams > 1) {
      // Where the head began before this block's ranges and goes on behind them, all of the block's workers have this head alone: they leave one part.
      const int first_worker = blockIdx.x * C::kTeams;
      if (!all && unit > 0 && unit + tiles < sp.units && ranges.of_position(head_end - cost + kHeadCost) < first_worker && ranges.of_position(head_end - 1) >= first_worker + C::kTeams) {
        constexpr int kEights = C::kRows / 8, kSteps = DP / 16;
        float4* sums = reinterpret_cast<float4*>(smem);  // [teams][eights][steps][32]
        float4* stats = sums + C::kTeams * kEights * kSteps * 32;
        copy_wait<0>();
        __syncthreads();  // the rings are free
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          const int eight = team * kEights + member * NR + n;
#pragma unroll
          for (int h = 0; h < 2; ++h)
            for (int x = 4; x < 32; x <<= 1) l[n][h] += __shfl_xor_sync(~0u, l[n][h], x);
#pragma unroll
          for (int t = 0; t < kSteps; ++t) sums[(eight * kSteps + t) * 32 + lane] = make_float4(o[t][n][0], o[t][n][1], o[t][n][2], o[t][n][3]);
          if (lane < 4) stats[eight * 4 + lane] = make_float4(m[n][0], m[n][1], l[n][0], l[n][1]);
        }
        __syncthreads();
        for (int i = warp; i < kEights * kSteps; i += kAttendWarps) {
          const int eight = i / kSteps, t = i - eight * kSteps;
          float4 st[C::kTeams], sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          float2 top = make_float2(-INFINITY, -INFINITY), total = make_float2(0.0f, 0.0f);
#pragma unroll
          for (int w = 0; w < C::kTeams; ++w) {
            st[w] = stats[(w * kEights + eight) * 4 + (lane & 3)];
            top = make_float2(fmaxf(top.x, st[w].x), fmaxf(top.y, st[w].y));
          }
#pragma unroll
          for (int w = 0; w < C::kTeams; ++w) {
            const float a = exp2_approx(st[w].x - (top.x == -INFINITY ? 0.0f : top.x)), c = exp2_approx(st[w].y - (top.y == -INFINITY ? 0.0f : top.y));
            const float4 v = sums[((w * kEights + eight) * kSteps + t) * 32 + lane];
            total = make_float2(fmaf(a, st[w].z, total.x), fmaf(c, st[w].w, total.y));
            sum = make_float4(fmaf(a, v.x, sum.x), fmaf(c, v.y, sum.y), fmaf(a, v.z, sum.z), fmaf(c, v.w, sum.w));
          }
          const int64_t at = 2 * (int64_t)first_worker * kEights + eight;
          if (16 * t < p.d) p.part_sums[(at * kSteps + t) * 32 + lane] = sum;
          if (t == 0 && lane < 4) p.part_stats[at * 4 + lane] = make_float4(top.x, top.y, total.x, total.y);
        }
        return;  // the range ends here
      }
    }
    const float v_scale = p.v_scale ? load_f32(p.v_scale + kv) : 1.0f;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const int eight = member * NR + n;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        for (int x = 4; x < 32; x <<= 1) l[n][h] += __shfl_xor_sync(~0u, l[n][h], x);
      if (all) {
        const Finish<F8> to(p, sp, b, kv, row0 + 8 * eight, v_scale, make_float2(l[n][0], l[n][1]));
        if (lane < 4) to.write_lse(p, make_float2(m[n][0], m[n][1]), make_float2(l[n][0], l[n][1]), C::kShift);
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) to.write(p, t, make_float4(o[t][n][0], o[t][n][1], o[t][n][2], o[t][n][3]));
      } else {
        float4* part = p.part_sums + ((slot * (C::kRows / 8) + eight) * (DP / 16)) * 32 + lane;
#pragma unroll
        for (int t = 0; t < DP / 16; ++t)
          if (16 * t < p.d) part[t * 32] = make_float4(o[t][n][0], o[t][n][1], o[t][n][2], o[t][n][3]);
        if (lane < 4) p.part_stats[(slot * (C::kRows / 8) + eight) * 4 + lane] = make_float4(m[n][0], m[n][1], l[n][0], l[n][1]);
      }
    }
    copy_wait<0>();
    team_sync<TEAM>(team);  // the ring is free for the next head
  }
}

// Adds up what the workers that shared a head left, and writes the rows that see nothing. A group of kWarps warps has one eight of rows and 32 of their
// elements; its warps take the parts in turn, each with a maximum of its own, and are joined through shared memory. One warp where a head has few parts, 16
// where few heads are in many (a warp per row of 128 elements took 16 us to add up 111 parts). Bound by the latency of four dependent loads.
constexpr int kJoinColumns = 2;  // of 16 elements

template <int kWarps>
struct JoinCfg {
  static constexpr int kThreads = kWarps == 1 ? 256 : 32 * kWarps, kGroups = kThreads / 32 / kWarps;
  static constexpr int kTake = kWarps == 16 ? 4 : 2;  // parts whose loads are in flight together
  static constexpr int kBlocksPerSm = kWarps == 16 ? 1 : 1024 / kThreads;
};

template <int DP, bool F8, int ROWS, int UNIT, int kWarps>
__global__ void __launch_bounds__(JoinCfg<kWarps>::kThreads, JoinCfg<kWarps>::kBlocksPerSm) paged_attention_join_kernel(const AttendArgs p, float shift) {
  constexpr int kEights = ROWS / 8, kSteps = DP / 16, kGroups = JoinCfg<kWarps>::kGroups, kTake = JoinCfg<kWarps>::kTake, T = AttendCfg<DP, F8, ROWS>::kTeams;
  __shared__ float4 s_stats[kWarps][4], s_sums[kWarps > 1 ? kWarps : 1][kJoinColumns][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, member = warp % kWarps;
  // Nothing is read before this, the lengths included: that the kernel in front has waited for who wrote them makes them visible to that kernel, not to this one
  // (read early they saved 0.5 to 1 us a call).
  griddep_wait();
  const int rows = p.queries * p.group.d, eights = rows < ROWS ? (rows + 7) / 8 : kEights, columns = (p.d + 16 * kJoinColumns - 1) / (16 * kJoinColumns);
  const int64_t items = (int64_t)p.spans * p.kv_heads * eights * columns;
  for (int64_t first = (int64_t)blockIdx.x * kGroups; first < items; first += (int64_t)gridDim.x * kGroups) {
    const int64_t item = first + warp / kWarps;
    if (item >= items) continue;  // a group is a warp, or the block
    const int64_t x0 = item / columns, at = x0 / eights;
    const int t0 = (int)(item - x0 * columns) * kJoinColumns, eight = (int)(x0 - at * eights), index = (int)(at / p.kv_heads), kv = (int)(at - (int64_t)index * p.kv_heads);
    const int b = p.row_tiles == 1 ? index : index / p.row_tiles, row0 = (index - b * p.row_tiles) * ROWS + 8 * eight;
    int4 sh = p.shares[at];  // asked for with the lengths; what a head without keys has there is not looked at
    const Span sp = span_of<ROWS, UNIT>(p, index);
    if (!sp.units) sh = make_int4(0, 1, 0, 0);
    // Parts of workers, but of the blocks between the first worker's and the last one's one part each.
    const int kept = T > 1 ? (sh.x / T + 1) * T - sh.x : 1, between = T > 1 ? sh.y / T - sh.x / T - 1 : 0;
    const int n = !sp.units ? 0 : between <= 0 ? sh.y - sh.x + 1 : kept + between + sh.y % T + 1;
    if (row0 >= rows || n == 1) continue;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    float4 acc[kJoinColumns];
#pragma unroll
    for (int t = 0; t < kJoinColumns; ++t) acc[t] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int x = member; x < n; x += kTake * kWarps) {
      float4 st[kTake], v[kTake][kJoinColumns];
#pragma unroll
      for (int y = 0; y < kTake; ++y) {  // all loads before the first use; those behind the last part read it again
        const int z = x + y * kWarps < n ? x + y * kWarps : x;
        const int worker = between <= 0 || z < kept ? sh.x + z : z < kept + between ? (sh.x / T + 1 + z - kept) * T : sh.y / T * T + z - kept - between;
        const int64_t slot = z == 0 ? (int64_t)sh.z : 2 * (int64_t)worker;  // all but the first worker of a head begin with it
        st[y] = p.part_stats[(slot * kEights + eight) * 4 + (lane & 3)];
#pragma unroll
        for (int t = 0; t < kJoinColumns; ++t) v[y][t] = p.part_sums[((slot * kEights + eight) * kSteps + (16 * (t0 + t) < p.d ? t0 + t : t0)) * 32 + lane];
      }
      float top[2] = {m[0], m[1]};
#pragma unroll
      for (int y = 0; y < kTake; ++y) {
        if (x + y * kWarps >= n) continue;
        top[0] = fmaxf(top[0], st[y].x), top[1] = fmaxf(top[1], st[y].y);
      }
      const float base[2] = {top[0] == -INFINITY ? 0.0f : top[0], top[1] == -INFINITY ? 0.0f : top[1]};
      const float keep[2] = {exp2_approx(m[0] - base[0]), exp2_approx(m[1] - base[1])};
#pragma unroll
      for (int h = 0; h < 2; ++h) l[h] *= keep[h], m[h] = top[h];
#pragma unroll
      for (int t = 0; t < kJoinColumns; ++t) acc[t].x *= keep[0], acc[t].y *= keep[1], acc[t].z *= keep[0], acc[t].w *= keep[1];
#pragma unroll
      for (int y = 0; y < kTake; ++y) {
        if (x + y * kWarps >= n) continue;
        const float w[2] = {exp2_approx(st[y].x - base[0]), exp2_approx(st[y].y - base[1])};
        l[0] = fmaf(w[0], st[y].z, l[0]), l[1] = fmaf(w[1], st[y].w, l[1]);
#pragma unroll
        for (int t = 0; t < kJoinColumns; ++t) {
          acc[t].x = fmaf(w[0], v[y][t].x, acc[t].x), acc[t].y = fmaf(w[1], v[y][t].y, acc[t].y);
          acc[t].z = fmaf(w[0], v[y][t].z, acc[t].z), acc[t].w = fmaf(w[1], v[y][t].w, acc[t].w);
        }
      }
    }
    if constexpr (kWarps > 1) {
      __syncthreads();
      if (lane < 4) s_stats[warp][lane] = make_float4(m[0], m[1], l[0], l[1]);
#pragma unroll
      for (int t = 0; t < kJoinColumns; ++t) s_sums[warp][t][lane] = acc[t];
      __syncthreads();
      if (member >= kJoinColumns) continue;  // a warp per 16 elements adds the warps up, in their order
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top[0] = fmaxf(top[0], s_stats[w][lane & 3].x), top[1] = fmaxf(top[1], s_stats[w][lane & 3].y);
      acc[0] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      l[0] = l[1] = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float4 st = s_stats[w][lane & 3], v = s_sums[w][member][lane];
        const float a = exp2_approx(st.x - (top[0] == -INFINITY ? 0.0f : top[0])), c = exp2_approx(st.y - (top[1] == -INFINITY ? 0.0f : top[1]));
        l[0] = fmaf(a, st.z, l[0]), l[1] = fmaf(c, st.w, l[1]);
        acc[0].x = fmaf(a, v.x, acc[0].x), acc[0].y = fmaf(c, v.y, acc[0].y), acc[0].z = fmaf(a, v.z, acc[0].z), acc[0].w = fmaf(c, v.w, acc[0].w);
      }
      m[0] = top[0], m[1] = top[1];
    }
    const Finish<F8> to(p, sp, b, kv, row0, p.v_scale ? load_f32(p.v_scale + kv) : 1.0f, make_float2(l[0], l[1]));
    if (lane < 4 && t0 == 0 && member == 0) to.write_lse(p, make_float2(m[0], m[1]), make_float2(l[0], l[1]), shift);
    if constexpr (kWarps > 1) {
      to.write(p, t0 + member, acc[0]);
    } else {
#pragma unroll
      for (int t = 0; t < kJoinColumns; ++t) to.write(p, t0 + t, acc[t]);
    }
  }
}

// Blocks of a call: as many as fit the device at once, or as the list can need.
template <int DP, bool F8, int ROWS>
static int attend_blocks(int64_t spans, int64_t kv_heads, int64_t entries) {
  using C = AttendCfg<DP, F8, ROWS>;
  const int64_t cap = (int64_t)sm_count() * C::kBlocksPerSm;
  const int64_t heads = spans * kv_heads, each = (entries + C::kKeys - 1) / C::kKeys + kHeadCost;
  if (heads >= cap * C::kTeams || each >= cap * C::kTeams || heads * each >= cap * C::kTeams) return (int)cap;
  return (int)((heads * each + C::kTeams - 1) / C::kTeams);
}

template <int DP, bool F8, int ROWS>
int64_t AttendCall<DP, F8, ROWS>::workspace(int64_t spans, int64_t kv_heads, int64_t entries) {
  using C = AttendCfg<DP, F8, ROWS>;
  return 2 * (int64_t)attend_blocks<DP, F8, ROWS>(spans, kv_heads, entries) * C::kTeams * C::kRows * (DP + 2) * 4 + spans * kv_heads * 16;
}

template <int DP, bool F8, int ROWS>
tf_status AttendCall<DP, F8, ROWS>::launch(AttendArgs p, void* workspace_at, int64_t workspace_bytes, cudaStream_t stream, const char* fn) {
  using C = AttendCfg<DP, F8, ROWS>;
  const int64_t need = workspace(p.spans, p.kv_heads, p.entries);
  if (need > workspace_bytes || !workspace_at)
    return fail(TF_ERR_WORKSPACE, "%s: the workspace needs %lld bytes, %lld were given", fn, (long long)need, (long long)workspace_bytes);
  auto kernel = paged_attention_kernel<DP, F8, ROWS>;
  static thread_local int configured_dev = -1;
  int dev = 0;
  TF_CUDA(cudaGetDevice(&dev));
  if (configured_dev != dev) {
    TF_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    configured_dev = dev;
  }
  p.whole_tiles = p.page.d % C::kKeys == 0;
  const int blocks = attend_blocks<DP, F8, ROWS>(p.spans, p.kv_heads, p.entries);
  const int64_t slots = 2 * (int64_t)blocks * C::kTeams, heads = (int64_t)p.spans * p.kv_heads;
  p.part_sums = static_cast<float4*>(workspace_at);
  p.part_stats = p.part_sums + slots * C::kRows * DP / 4;
  p.shares = reinterpret_cast<int4*>(p.part_stats + slots * C::kRows / 2);
  TF_CUDA(launch_dependent(true, kernel, dim3((unsigned)blocks), dim3(kAttendThreads), C::kSmem, stream, p));
  const int64_t rows = (int64_t)p.queries * p.group.d, eights = ((rows < C::kRows ? rows : C::kRows) + 7) / 8;
  const int64_t items = heads * eights * ((p.d + 16 * kJoinColumns - 1) / (16 * kJoinColumns)), most = (int64_t)sm_count() * 16;
  auto join = [&](auto form) -> cudaError_t {
    constexpr int kWarps = decltype(form)::value;
    using J = JoinCfg<kWarps>;
    const int64_t groups = (items + J::kGroups - 1) / J::kGroups;
    return launch_dependent(true, paged_attention_join_kernel<DP, F8, C::kRows, C::kKeys, kWarps>, dim3((unsigned)(groups < most ? groups : most)), dim3(J::kThreads), 0, stream, p,
                            C::kShift);
  };
  // Workers over heads are the parts of a head on average, and over heads and teams where blocks join their own. 16 warps only where all items are resident
  // at once (40 rows of 120 heads, ten parts each: 69 us with 16 warps, 42 with four; two sequences of 131072, 111 parts of 16 heads: 116 us with 16, 125 with four).
  const int64_t workers = (int64_t)blocks * C::kTeams, parts = workers / heads <= 2 * C::kTeams ? workers / heads : workers / heads / C::kTeams + C::kTeams;
  if (parts > 8 && items <= 2 * (int64_t)sm_count())
    TF_CUDA(join(std::integral_constant<int, 16>{}));
  else if (parts > 4)
    TF_CUDA(join(std::integral_constant<int, 4>{}));
  else
    TF_CUDA(join(std::integral_constant<int, 1>{}));
  return TF_OK;
}

}  // namespace tf
