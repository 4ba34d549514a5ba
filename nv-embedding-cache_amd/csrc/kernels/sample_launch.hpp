// sample_launch.hpp -- host launcher of the token sampling kernel (sample.hip).
//
// Every pointer is device memory; shapes and types are checked by the caller (sample.cpp).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace nve_amd {

struct Sample {
  int64_t rows, vocab;
  int32_t dtype;
  const uint8_t* logits;
  int64_t row_stride;  // in elements
  const float* u;
  // [rows], or null: the same for all rows
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all;
  int32_t top_k_all;
  float top_p_all, min_p_all;
  int64_t* tokens;
};

size_t sample_workspace(const Sample& a);
hipError_t launch_sample(const Sample& a, void* workspace, hipStream_t stream);

}  // namespace nve_amd
