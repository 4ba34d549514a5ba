// sample.cpp -- token sampling: argument checks and launch (kernels/sample.hip).
//
// Everything the host can see is checked here; limits of single rows lie in device memory, and the
// kernels take each value of them (see nve_amd_sample_t).
#include "sample.hpp"

#include "dtypes.hpp"
#include "kernels/sample_launch.hpp"
#include "runtime.hpp"

namespace nve_amd {

namespace {

Sample sample_of(const nve_amd_sample_t* p) {
  NVE_CHECK_ARG(p != nullptr, "call must not be NULL");
  NVE_CHECK_ARG(p->num_rows >= 0 && p->num_rows <= (1 << 30), "Invalid num_rows ", p->num_rows);
  NVE_CHECK_ARG(p->vocab_size >= 1 && p->vocab_size <= (1 << 30), "vocab_size must be in [1, 2^30] (got ",
                p->vocab_size, ")");
  const int dt = (int)p->dtype;
  NVE_CHECK_ARG(dt == kF32 || dt == kF16 || dt == kBF16, "logits must be float32, float16 or bfloat16 (got type ", dt,
                ")");
  if (p->num_rows > 0) NVE_CHECK_ARG(p->logits && p->u && p->tokens, "logits, u and tokens must not be NULL");
  // a NaN fails these too
  if (!p->temperatures) NVE_CHECK_ARG(p->temperature >= 0, "temperature must not be negative (got ", p->temperature, ")");
  if (!p->top_ks) NVE_CHECK_ARG(p->top_k >= 0, "top_k must not be negative (got ", p->top_k, ")");
  if (!p->top_ps) NVE_CHECK_ARG(p->top_p >= 0, "top_p must not be negative (got ", p->top_p, ")");
  if (!p->min_ps) NVE_CHECK_ARG(p->min_p >= 0 && p->min_p <= 1, "min_p must be in [0, 1] (got ", p->min_p, ")");
  Sample a{};
  a.rows = p->num_rows;
  a.vocab = p->vocab_size;
  a.dtype = dt;
  a.logits = static_cast<const uint8_t*>(p->logits);
  a.row_stride = p->row_stride;
  a.u = p->u;
  a.temperature = p->temperatures;
  a.top_k = p->top_ks;
  a.top_p = p->top_ps;
  a.min_p = p->min_ps;
  a.temperature_all = p->temperature;
  a.top_k_all = p->top_k;
  a.top_p_all = p->top_p;
  a.min_p_all = p->min_p;
  a.tokens = p->tokens;
  return a;
}

}  // namespace

size_t sample_workspace_bytes(const nve_amd_sample_t* call) { return sample_workspace(sample_of(call)); }

void sample_run(const nve_amd_sample_t* call, void* ws, size_t ws_bytes, hipStream_t s) {
  const Sample a = sample_of(call);
  const size_t need = sample_workspace(a);
  if (need > 0) {
    NVE_CHECK_ARG(ws != nullptr && ws_bytes >= need, "Workspace too small: ", ws_bytes, " bytes, ", need, " needed");
    NVE_CHECK_ARG(reinterpret_cast<uintptr_t>(ws) % 16 == 0, "The workspace must be 16-byte aligned");
  }
  NVE_HIP(launch_sample(a, ws, s));
}

}  // namespace nve_amd
