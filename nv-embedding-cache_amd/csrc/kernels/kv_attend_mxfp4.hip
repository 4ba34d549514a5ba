// kv_attend_mxfp4.hip -- attention over pages of 4-bit values (kv_attend.cuh).
#include "kv_attend.cuh"

namespace nve_amd {

hipError_t launch_kv_attend_mxfp4(const KvAttend& a, void* workspace, hipStream_t stream) {
  return a.dtype == kF16 ? launch_types<kF16, kMXFP4>(a, workspace, stream)
                         : launch_types<kBF16, kMXFP4>(a, workspace, stream);
}

}  // namespace nve_amd
