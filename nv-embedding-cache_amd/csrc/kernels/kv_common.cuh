// kv_common.cuh -- device helpers shared by the paged key-value cache's kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../dtypes.hpp"
#include "kv_launch.hpp"

namespace nve_amd {

// Element types of queries, outputs and unscaled pages.
template <int DT>
struct KvElem;
template <>
struct KvElem<kF32> {
  using type = float;
};
template <>
struct KvElem<kF16> {
  using type = _Float16;
};
template <>
struct KvElem<kBF16> {
  using type = __bf16;
};
template <int DT>
using kv_elem = typename KvElem<DT>::type;

// The page of slot t of a sequence whose table row is `table`, or -1: absent.
__device__ __forceinline__ int64_t kv_page(const KvPages& c, const int32_t* table, int64_t t) {
  const int64_t p = table[t >> c.page_bits];
  return p >= 0 && p < c.num_pages ? p : -1;
}

// Row number of a slot of `head` in [num_pages, heads, page].
__device__ __forceinline__ int64_t kv_row(const KvPages& c, int64_t page, int head, int64_t t) {
  return ((page * c.heads + head) << c.page_bits) + (t & (c.page - 1));
}

// The slots of sequence s that count.
__device__ __forceinline__ int64_t kv_length(const int32_t* lengths, int64_t s, int64_t max_length) {
  const int64_t n = lengths[s];
  return n < 0 ? 0 : n < max_length ? n : max_length;
}

// x of the lanes up to and including this one, added; every lane of the wave is on.
// Row shifts by 1, 2, 4 and 8, then each row's last lane to the rows behind it.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
  asm volatile("" : "+v"(x));  // not moved under a condition, where some lanes are off
  return x;
}

}  // namespace nve_amd
