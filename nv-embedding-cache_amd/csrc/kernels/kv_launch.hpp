// kv_launch.hpp -- host launchers of the paged key-value cache's kernels
// (kv_append.hip, kv_attend.hip, kv_attend_mxfp4.hip, kv_evict.hip).
//
// Every pointer is device memory; shapes, types and strides are checked by the
// caller (kv_cache.cpp).  Values read from device memory (slots, positions,
// page ids, lengths) are checked against their bounds in the kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../dtypes.hpp"

namespace nve_amd {

// Bytes of a head's row.
inline constexpr int kv_row_bytes(int dtype, int dim) { return dtype == kMXFP4 ? dim / 2 : dim * value_elem_bytes(dtype); }

// The pages: k and v [num_pages, heads, page, dim] of dtype, the rest [num_pages, heads, page]
// (kMXFP4: the scales are [num_pages, heads, page, dim / 32] bytes).
struct KvPages {
  uint8_t* k;
  uint8_t* v;
  void* k_scale;
  void* v_scale;
  float* weights;
  int32_t* index;
  int64_t num_pages;
  int32_t heads, page, page_bits, dim, dtype;
};

// Rows of `heads` heads per token, strides in elements.
struct KvRows {
  const uint8_t* p;
  int64_t token_stride, head_stride;
};

struct KvAppend {
  KvPages pages;
  int64_t tokens;
  const int64_t* slots;
  int32_t dtype;
  KvRows k, v, q;
  uint8_t* q_out;
  int64_t q_out_token_stride, q_out_head_stride;
  int32_t q_heads;
  const int32_t* index;
  const int32_t* positions;
  int64_t axis_stride;
  const float* cos_sin;
  int64_t max_position;
  int32_t rot, interleaved, axes;
  int32_t ends[4];  // the first pair past each axis
  const uint8_t* q_norm;  // [dim] of dtype, or null: no norm
  const uint8_t* k_norm;
  double eps, inverse_dim;
};

struct KvAttend {
  KvPages pages;
  int64_t seqs;
  int32_t q_heads, dtype;
  KvRows q;
  uint8_t* out;
  int64_t out_seq_stride, out_head_stride;
  float* lse;  // may be null
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* lengths;
  int64_t max_length;  // lengths above it count as it
  float scale;
  int32_t accumulate;
};

struct KvEvict {
  KvPages pages;
  int64_t seqs;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* lengths;
  int32_t* new_lengths;
  int64_t max_length;
  int64_t budget, sinks, recent;
};

hipError_t launch_kv_append(const KvAppend& a, hipStream_t stream);
size_t kv_attend_workspace(const KvAttend& a);
hipError_t launch_kv_attend(const KvAttend& a, void* workspace, hipStream_t stream);
hipError_t launch_kv_attend_mxfp4(const KvAttend& a, void* workspace, hipStream_t stream);  // of launch_kv_attend
size_t kv_evict_workspace(const KvEvict& a);
hipError_t launch_kv_evict(const KvEvict& a, void* workspace, hipStream_t stream);

}  // namespace nve_amd
