// kv_append.hip -- new tokens enter the paged key-value cache: rotary positions
// on queries and keys, keys and values written to their slots.
//
// One wave per head row: lane l holds values l, l + 64, ...; a rotated value
// reads its pair's other value itself, so nothing crosses lanes but an e4m3
// row's largest magnitude.
#include "kv_common.cuh"

namespace nve_amd {

namespace {

constexpr int kRowsPerBlock = 4;  // waves
constexpr int kMaxPer = 4;        // values per lane: head_dim <= 256

// Value d of a head row of token t, rotated; f32 products and sum rounded one by one.
template <typename T>
__device__ __forceinline__ float rotated(const KvAppend& a, const T* row, int64_t t, int d) {
  const float x = (float)row[d];
  if (d >= a.rot) return x;
  const int half = a.rot >> 1;
  const int pair = a.interleaved ? d >> 1 : (d < half ? d : d - half);
  const bool first = a.interleaved ? (d & 1) == 0 : d < half;
  const int other = a.interleaved ? d ^ 1 : (first ? d + half : d - half);
  int axis = 0;
  while (axis + 1 < a.axes && pair >= a.ends[axis]) ++axis;
  const int64_t p = a.positions[axis * a.axis_stride + t];
  if (p < 0 || p >= a.max_position) return x;
  const float* cs = a.cos_sin + p * a.rot;
  const float c = cs[pair], s = cs[pair + half], y = (float)row[other];
  return first ? x * c - y * s : x * c + y * s;
}

template <int DT, bool E4M3>
__global__ __launch_bounds__(64 * kRowsPerBlock) void kv_append_kernel(const KvAppend a) {
  using T = kv_elem<DT>;
  const int lane = threadIdx.x & 63;
  const int rows = a.q_heads + 2 * a.pages.heads;
  const int64_t r = (int64_t)blockIdx.x * kRowsPerBlock + (threadIdx.x >> 6);
  const int64_t t = r / rows;
  if (t >= a.tokens) return;
  int head = (int)(r - t * rows);
  const int dim = a.pages.dim;
  if (head < a.q_heads) {
    const T* row = reinterpret_cast<const T*>(a.q.p) + t * a.q.token_stride + head * a.q.head_stride;
    T* out = reinterpret_cast<T*>(a.q_out) + t * a.q_out_token_stride + head * a.q_out_head_stride;
    float x[kMaxPer];
#pragma unroll
    for (int i = 0; i < kMaxPer; ++i)
      if (lane + 64 * i < dim) x[i] = rotated(a, row, t, lane + 64 * i);
    // q_out may be q: every lane's values are read before the first is written
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < kMaxPer; ++i)
      if (lane + 64 * i < dim) out[lane + 64 * i] = (T)x[i];
    return;
  }
  head -= a.q_heads;
  const bool value = head >= a.pages.heads;
  if (value) head -= a.pages.heads;
  const int64_t slot = a.slots[t];
  if (slot < 0 || slot >> a.pages.page_bits >= a.pages.num_pages) return;
  const int64_t at = kv_row(a.pages, slot >> a.pages.page_bits, head, slot);
  const KvRows& in = value ? a.v : a.k;
  const T* row = reinterpret_cast<const T*>(in.p) + t * in.token_stride + head * in.head_stride;
  uint8_t* pages = value ? a.pages.v : a.pages.k;
  float x[kMaxPer];
#pragma unroll
  for (int i = 0; i < kMaxPer; ++i) {
    const int d = lane + 64 * i;
    x[i] = d >= dim ? 0.0f : value ? (float)row[d] : rotated(a, row, t, d);
  }
  if constexpr (E4M3) {
    // the largest magnitude by its bits, so that a NaN is the largest of all
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kMaxPer; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m));
    const float scale = __uint_as_float(max(top, __float_as_uint(1e-30f))) / 448.0f;
#pragma unroll
    for (int i = 0; i < kMaxPer; ++i)
      if (lane + 64 * i < dim)
        pages[at * dim + lane + 64 * i] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[i] / scale, 0.0f, 0, false);
    if (lane == 0) (value ? a.pages.v_scale : a.pages.k_scale)[at] = scale;
  } else {
    T* out = reinterpret_cast<T*>(pages) + at * dim;
#pragma unroll
    for (int i = 0; i < kMaxPer; ++i)
      if (lane + 64 * i < dim) out[lane + 64 * i] = (T)x[i];
  }
  if (lane == 0 && value) {
    if (a.pages.index) a.pages.index[at] = a.index ? a.index[t] : a.positions ? a.positions[t] : 0;
    if (a.pages.weights) a.pages.weights[at] = 0.0f;
  }
}

}  // namespace

hipError_t launch_kv_append(const KvAppend& a, hipStream_t stream) {
  const int64_t rows = a.tokens * (a.q_heads + 2 * a.pages.heads);
  if (rows == 0) return hipSuccess;
  const dim3 grid((unsigned)((rows + kRowsPerBlock - 1) / kRowsPerBlock)), block(64 * kRowsPerBlock);
  const bool q8 = a.pages.dtype == kE4M3;
  switch (a.dtype) {
    case kF32: kv_append_kernel<kF32, false><<<grid, block, 0, stream>>>(a); break;
    case kF16:
      if (q8) kv_append_kernel<kF16, true><<<grid, block, 0, stream>>>(a);
      else kv_append_kernel<kF16, false><<<grid, block, 0, stream>>>(a);
      break;
    case kBF16:
      if (q8) kv_append_kernel<kBF16, true><<<grid, block, 0, stream>>>(a);
      else kv_append_kernel<kBF16, false><<<grid, block, 0, stream>>>(a);
      break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace nve_amd
