// nve_sample_ops.cpp -- the nve_ops torch library's token sampling (HIP tensors), calling
// libnve_amd.so's C ABI (nve_amd_sample) directly:
//
//   sample_tokens   (schema below)
//
// Shapes, types and devices are checked here, the rest by the C ABI; work runs on the current
// stream, the workspace comes from torch's allocator.  There is no gradient, and logits that ask
// for one are refused.
#include <ATen/DeviceGuard.h>
#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <cstdint>
#include <optional>
#include <string>

#include "nve_amd_ext.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

void check_status(nve_status_t st) {
  if (st == NVE_SUCCESS) return;
  const char* m = nullptr;
  nve_get_last_error(&m);
  const std::string what = m ? m : "no message";
  TORCH_CHECK_VALUE(st != NVE_ERROR_INVALID_ARGUMENT, "nve_ops: invalid argument: ", what);
  TORCH_CHECK(false, "nve_ops: status ", (int)st, ": ", what);
}

// A value for each row.
template <typename T>
const T* of_rows(const OptTensor& t, const Tensor& logits, at::ScalarType type, const char* name) {
  if (!t.has_value() || !t->defined()) return nullptr;
  TORCH_CHECK_VALUE(t->device() == logits.device(), "nve_ops: ", name, " is on ", t->device(), ", the logits on ",
                    logits.device());
  TORCH_CHECK_TYPE(t->scalar_type() == type, "nve_ops: ", name, " must be ", type, ", got ", t->scalar_type());
  TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == logits.size(0) && t->is_contiguous(), "nve_ops: ", name,
                    " must be contiguous and [", logits.size(0), "], got ", t->sizes());
  return static_cast<const T*>(t->data_ptr());
}

Tensor sample_tokens(const Tensor& logits, const Tensor& u, const OptTensor& temperatures, const OptTensor& top_ks,
                     const OptTensor& top_ps, const OptTensor& min_ps, double temperature, int64_t top_k, double top_p,
                     double min_p) {
  const at::DeviceGuard guard(logits.device());
  TORCH_CHECK_VALUE(logits.dim() == 2, "nve_ops: logits must be [rows, vocabulary], got ", logits.sizes());
  TORCH_CHECK_VALUE(logits.stride(1) == 1 || logits.size(1) <= 1 || logits.size(0) == 0,
                    "nve_ops: the last dimension of logits must be contiguous");
  TORCH_CHECK(!(logits.requires_grad() && at::GradMode::is_enabled()),
              "nve_ops: logits asks for a gradient, and sampling has none (use torch.no_grad())");
  TORCH_CHECK_VALUE(top_k <= INT32_MAX, "nve_ops: top_k is too large: ", top_k);
  nve_amd_sample_t c{};
  switch (logits.scalar_type()) {
    case at::kFloat: c.dtype = NVE_DTYPE_FLOAT32; break;
    case at::kHalf: c.dtype = NVE_DTYPE_FLOAT16; break;
    case at::kBFloat16: c.dtype = NVE_DTYPE_BFLOAT16; break;
    default: TORCH_CHECK_TYPE(false, "nve_ops: logits cannot be ", logits.scalar_type());
  }
  c.num_rows = logits.size(0);
  c.vocab_size = logits.size(1);
  c.logits = logits.data_ptr();
  c.row_stride = logits.stride(0);
  c.u = of_rows<float>(u, logits, at::kFloat, "u");
  c.temperatures = of_rows<float>(temperatures, logits, at::kFloat, "temperature");
  c.top_ks = of_rows<int32_t>(top_ks, logits, at::kInt, "top_k");
  c.top_ps = of_rows<float>(top_ps, logits, at::kFloat, "top_p");
  c.min_ps = of_rows<float>(min_ps, logits, at::kFloat, "min_p");
  c.temperature = (float)temperature;
  c.top_k = (int32_t)(top_k < 0 ? -1 : top_k);
  c.top_p = (float)top_p;
  c.min_p = (float)min_p;
  Tensor tokens = at::empty({logits.size(0)}, logits.options().dtype(at::kLong));
  c.tokens = static_cast<int64_t*>(tokens.data_ptr());
  uint64_t need = 0;
  check_status(nve_amd_sample_workspace_size(&c, &need));
  Tensor ws;
  if (need > 0) ws = at::empty({(int64_t)need}, logits.options().dtype(at::kByte));
  check_status(nve_amd_sample(&c, need > 0 ? ws.data_ptr() : nullptr, need,
                              c10::hip::getCurrentHIPStream(logits.get_device()).stream()));
  return tokens;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(nve_ops, m) {
  m.def(
      "sample_tokens(Tensor logits, Tensor u, Tensor? temperatures, Tensor? top_ks, Tensor? top_ps, Tensor? min_ps, "
      "float temperature, int top_k, float top_p, float min_p) -> Tensor");
}

TORCH_LIBRARY_IMPL(nve_ops, CUDA, m) { m.impl("sample_tokens", &sample_tokens); }
