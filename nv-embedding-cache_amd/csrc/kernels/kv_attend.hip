// kv_attend.hip -- attention of one new token per sequence over its pages.
//
// One workgroup per (sequence, query head).  Tiles of 256 slots: a thread takes
// a slot's score, the workgroup the running maximum and sum of the softmax, and
// then a thread takes one value of the output row over the tile's slots.
#include <math.h>

#include "kv_common.cuh"

namespace nve_amd {

namespace {

constexpr int kTile = 256;
constexpr float kLog2e = 1.4426950408889634f;

template <int DT, bool E4M3>
__device__ __forceinline__ float load_value(const uint8_t* p, int64_t i) {
  if constexpr (E4M3) return __builtin_amdgcn_cvt_f32_fp8((int)p[i], 0);
  else return (float)reinterpret_cast<const kv_elem<DT>*>(p)[i];
}

template <int DT, bool E4M3>
__global__ __launch_bounds__(kTile) void kv_attend_kernel(const KvAttend a, float* logits, float* lse) {
  using T = kv_elem<DT>;
  __shared__ float q[256];
  __shared__ float p[kTile];
  __shared__ int64_t row[kTile];
  __shared__ float red[8];
  const int tid = threadIdx.x, dim = a.pages.dim;
  const int64_t s = blockIdx.x;
  const int qh = blockIdx.y, head = qh / (a.q_heads / a.pages.heads);
  const int64_t len = kv_length(a.lengths, s, a.max_length);
  const T* qrow = reinterpret_cast<const T*>(a.q.p) + s * a.q.token_stride + qh * a.q.head_stride;
  if (tid < dim) q[tid] = (float)qrow[tid];
  __syncthreads();
  float m = -INFINITY, l = 0.0f, acc = 0.0f;
  for (int64_t t0 = 0; t0 < len; t0 += kTile) {
    const int64_t t = t0 + tid;
    float x = -INFINITY;
    int64_t at = -1;
    if (t < len) {
      const int64_t page = kv_page(a.pages, a.tables + s * a.table_stride, t);
      if (page >= 0) {
        at = kv_row(a.pages, page, head, t);
        float dot = 0.0f;
        for (int d = 0; d < dim; ++d) dot = fmaf(q[d], load_value<DT, E4M3>(a.pages.k, at * dim + d), dot);
        if constexpr (E4M3) dot *= a.pages.k_scale[at];
        x = dot * a.scale;
      }
      if (logits) logits[(s * a.q_heads + qh) * a.max_length + t] = x;
    }
    row[tid] = at;
    const float wm = wave_max(x);
    if ((tid & 63) == 0) red[tid >> 6] = wm;
    __syncthreads();
    const float top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float nm = fmaxf(m, top);
    const float base = nm == -INFINITY ? 0.0f : nm;  // nothing but -infinity so far
    const float e = exp2f((x - base) * kLog2e);
    float w = e;
    if constexpr (E4M3)
      if (at >= 0) w *= a.pages.v_scale[at];
    p[tid] = w;
    const float ws = wave_sum(e);
    if ((tid & 63) == 0) red[4 + (tid >> 6)] = ws;
    __syncthreads();
    const float alpha = exp2f((m - base) * kLog2e);
    l = l * alpha + red[4] + red[5] + red[6] + red[7];
    acc *= alpha;
    m = nm;
    if (tid < dim) {
      const int n = (int)(len - t0 < kTile ? len - t0 : kTile);
      for (int j = 0; j < n; ++j)
        if (row[j] >= 0) acc = fmaf(p[j], load_value<DT, E4M3>(a.pages.v, row[j] * dim + tid), acc);
    }
    __syncthreads();
  }
  if (tid < dim) {
    T* out = reinterpret_cast<T*>(a.out) + s * a.out_seq_stride + qh * a.out_head_stride;
    out[tid] = (T)(l == 0.0f ? 0.0f : acc / l);  // no slot has a score above -infinity
  }
  if (tid == 0 && lse) lse[s * a.q_heads + qh] = m + logf(l);
}

// weights[slot] += sum over the group's query heads of exp(x - lse)
__global__ __launch_bounds__(kTile) void kv_weights_kernel(const KvAttend a, const float* logits, const float* lse) {
  const int64_t s = blockIdx.y;
  const int head = blockIdx.z, group = a.q_heads / a.pages.heads;
  const int64_t t = (int64_t)blockIdx.x * kTile + threadIdx.x;
  if (t >= kv_length(a.lengths, s, a.max_length)) return;
  const int64_t page = kv_page(a.pages, a.tables + s * a.table_stride, t);
  if (page < 0) return;
  float w = 0.0f;
  for (int g = 0; g < group; ++g) {
    const int64_t qh = s * a.q_heads + head * group + g;
    const float all = lse[qh];
    if (all != -INFINITY) w += exp2f((logits[qh * a.max_length + t] - all) * kLog2e);
  }
  a.pages.weights[kv_row(a.pages, page, head, t)] += w;
}

}  // namespace

size_t kv_attend_workspace(const KvAttend& a) {
  return a.accumulate ? (size_t)(a.seqs * a.q_heads) * 4 * (size_t)(a.max_length + 1) : 0;
}

hipError_t launch_kv_attend(const KvAttend& a, void* workspace, hipStream_t stream) {
  if (a.seqs == 0 || a.q_heads == 0) return hipSuccess;
  float* logits = a.accumulate ? static_cast<float*>(workspace) : nullptr;
  float* lse = a.lse ? a.lse : a.accumulate ? logits + a.seqs * a.q_heads * a.max_length : nullptr;
  const dim3 grid((unsigned)a.seqs, (unsigned)a.q_heads);
  const bool q8 = a.pages.dtype == kE4M3;
  switch (a.dtype) {
    case kF32: kv_attend_kernel<kF32, false><<<grid, kTile, 0, stream>>>(a, logits, lse); break;
    case kF16:
      if (q8) kv_attend_kernel<kF16, true><<<grid, kTile, 0, stream>>>(a, logits, lse);
      else kv_attend_kernel<kF16, false><<<grid, kTile, 0, stream>>>(a, logits, lse);
      break;
    case kBF16:
      if (q8) kv_attend_kernel<kBF16, true><<<grid, kTile, 0, stream>>>(a, logits, lse);
      else kv_attend_kernel<kBF16, false><<<grid, kTile, 0, stream>>>(a, logits, lse);
      break;
    default: return hipErrorInvalidValue;
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !a.accumulate || a.max_length == 0) return e;
  const dim3 wgrid((unsigned)((a.max_length + kTile - 1) / kTile), (unsigned)a.seqs, (unsigned)a.pages.heads);
  kv_weights_kernel<<<wgrid, kTile, 0, stream>>>(a, logits, lse);
  return hipGetLastError();
}

}  // namespace nve_amd
