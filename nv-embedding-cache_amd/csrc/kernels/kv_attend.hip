// kv_attend.hip -- attention over pages of f32, f16, bf16 and e4m3 (kv_attend.cuh).
#include "kv_attend.cuh"

namespace nve_amd {

size_t kv_attend_workspace(const KvAttend& a) { return a.seqs == 0 ? 0 : layout_of(a, nullptr).bytes; }

hipError_t launch_kv_attend(const KvAttend& a, void* workspace, hipStream_t stream) {
  if (a.seqs == 0) return hipSuccess;
  if (a.pages.dtype == kMXFP4) return launch_kv_attend_mxfp4(a, workspace, stream);
  const bool q8 = a.pages.dtype == kE4M3;
  switch (a.dtype) {
    case kF32: return launch_types<kF32, kF32>(a, workspace, stream);
    case kF16: return q8 ? launch_types<kF16, kE4M3>(a, workspace, stream) : launch_types<kF16, kF16>(a, workspace, stream);
    case kBF16:
      return q8 ? launch_types<kBF16, kE4M3>(a, workspace, stream) : launch_types<kBF16, kBF16>(a, workspace, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace nve_amd
