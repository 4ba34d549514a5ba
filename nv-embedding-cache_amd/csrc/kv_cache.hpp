// kv_cache.hpp -- the paged key-value cache's operators: argument checks and
// launches (kv_cache.cpp) behind the nve_amd_kv_* entry points.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/nve_amd_ext.h"

namespace nve_amd {

void kv_append_run(const nve_amd_kv_pages_t* pages, const nve_amd_kv_append_t* call, hipStream_t s);
void kv_append_norm_run(const nve_amd_kv_pages_t* pages, const nve_amd_kv_append_t* call,
                        const nve_amd_kv_norm_t* norm, hipStream_t s);
size_t kv_attend_workspace_bytes(const nve_amd_kv_pages_t* pages, const nve_amd_kv_attend_t* call);
void kv_attend_run(const nve_amd_kv_pages_t* pages, const nve_amd_kv_attend_t* call, void* ws, size_t ws_bytes,
                   hipStream_t s);
size_t kv_evict_workspace_bytes(const nve_amd_kv_pages_t* pages, const nve_amd_kv_evict_t* call);
void kv_evict_run(const nve_amd_kv_pages_t* pages, const nve_amd_kv_evict_t* call, void* ws, size_t ws_bytes,
                  hipStream_t s);

}  // namespace nve_amd
