// What the entry point of paged attention hands to the kernels (paged_attention.cuh), which are built in files of their own.
#pragma once

#include <cuda_bf16.h>

#include "paged_cache.h"

namespace tf {

struct AttendArgs {
  const uint8_t* k;
  const uint8_t* v;
  const float* k_scale;
  const float* v_scale;
  int64_t stride_page, stride_head, stride_slot;  // bytes
  int pages, kv_heads, d;
  Divisor page;
  bool whole_tiles;  // the page size is a multiple of the kernel's tile
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  float* lse;
  int64_t q_ldt, q_ldh, out_ldt, out_ldh;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* lengths;
  const int32_t* counts;
  int entries;  // what a table can name
  int spans;    // sequences x row tiles
  int queries, q_heads, row_tiles, window;
  Divisor group;
  float scale_log2;
  float4* part_sums;   // [2 * workers][rows / 8][elements / 16][32 lanes]: of a worker's first head, and of its last
  float4* part_stats;  // [2 * workers][rows / 8][4]: two rows' maxima and sums
  int4* shares;        // [spans * kv_heads]: the first and the last worker of a head, and the first one's slot
};

// The kernels for heads of up to DP elements, a bf16 or e4m3 cache and tiles of ROWS query rows. Defined in one object each: the workspace and the
// launch have to agree.
template <int DP, bool F8, int ROWS>
struct AttendCall {
  static int64_t workspace(int64_t spans, int64_t kv_heads, int64_t entries);
  static tf_status launch(AttendArgs p, void* workspace, int64_t workspace_bytes, cudaStream_t stream, const char* fn);
};

}  // namespace tf
