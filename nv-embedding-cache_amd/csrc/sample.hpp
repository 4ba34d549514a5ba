// sample.hpp -- token sampling: argument checks and launch (sample.cpp) behind nve_amd_sample.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/nve_amd_ext.h"

namespace nve_amd {

size_t sample_workspace_bytes(const nve_amd_sample_t* call);
void sample_run(const nve_amd_sample_t* call, void* ws, size_t ws_bytes, hipStream_t s);

}  // namespace nve_amd
