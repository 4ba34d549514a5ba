// kv_append.hip -- new tokens enter the paged key-value cache: rotary positions
// on queries and keys, keys and values written to their slots.
//
// Every value is read and written once, with 3 flops a rotated value: bound by
// the bytes.  kv_append_kernel: a head row is a group of lanes (a power of two),
// 16 values a lane.  A lane that rotates has 8 pairs, both values of each, so
// that nothing crosses lanes but an e4m3 row's largest magnitude: values 8 j ..
// and rot / 2 + 8 j .. of the row, or (pairs of neighbours) 16 j ..; the lanes
// behind them have 16 unrotated values.  A workgroup has whole tokens: it brings
// their cosines and sines into shared memory once for all their heads, while the
// first rows' loads are under way.
// Several tokens a workgroup once there are 2,048 workgroups: 9,000 tokens into e4m3
// 51 -> 42 us.  Measured: 16,001 f16 tokens of 32 query and 8 key heads of 128 values
// 83 to 92 us (4.4 to 4.8 TB/s; a large copy 4.7); 9,000 bf16 tokens of 96 values
// into e4m3 42 to 44 us (3.6 TB/s; 6 of 8 lanes a row work); a step of 64
// tokens 4.8 us, the chain position, cosine, shared memory, store.
// kv_append_any_kernel, for rows that start off 16 bytes and for rotated widths
// that are no multiple of 16: one value of a row per lane and step (409 us for the
// 16,001 tokens above).
#include <algorithm>

#include "kv_common.cuh"

namespace nve_amd {

namespace {

using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
using u32x2 = __attribute__((ext_vector_type(2))) uint32_t;
using f32x4 = __attribute__((ext_vector_type(4))) float;

// The largest magnitude by its bits, so that a NaN is the largest of all.
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ float e4m3_scale(uint32_t top) {
  return __uint_as_float(max(top, __float_as_uint(1e-30f))) / 448.0f;
}

__device__ __forceinline__ void write_slot(const KvAppend& a, int64_t t, int64_t at) {
  if (a.pages.index) a.pages.index[at] = a.index ? a.index[t] : a.positions ? a.positions[t] : 0;
  if (a.pages.weights) a.pages.weights[at] = 0.0f;
}

// The row of [pages, heads, page] that token t's head goes to, or -1.
__device__ __forceinline__ int64_t row_of(const KvAppend& a, int64_t t, int head) {
  const int64_t slot = a.slots[t], page = slot >> a.pages.page_bits;
  if (slot < 0 || page >= a.pages.num_pages) return -1;
  return kv_row(a.pages, page, head, slot);
}

__device__ __forceinline__ int axis_of(const KvAppend& a, int pair) {
  int axis = 0;
  while (axis + 1 < a.axes && pair >= a.ends[axis]) ++axis;
  return axis;
}

// ---------------------------------------------------------------------------
// 16 values a lane
// ---------------------------------------------------------------------------
constexpr int kThreads = 256;
constexpr int kMaxTable = 2048;  // cosines and sines in shared memory

// 8 values of a row, as they lie in memory: from, widened and (rounded) back.
template <int DT>
struct Eight {
  static constexpr int kWords = DT == kF32 ? 2 : 1;
  u32x4 w[kWords];
  __device__ __forceinline__ void load(const uint8_t* p) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = reinterpret_cast<const u32x4*>(p)[i];
  }
  __device__ __forceinline__ void get(float* x) const {
    using T = kv_elem<DT>;
    T v[8];
    __builtin_memcpy(v, w, sizeof v);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
  }
  static __device__ __forceinline__ void store(uint8_t* p, const float* x) {
    using T = kv_elem<DT>;
    T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (T)x[i];
    u32x4 w[kWords];
    __builtin_memcpy(w, v, sizeof v);
#pragma unroll
    for (int i = 0; i < kWords; ++i) reinterpret_cast<u32x4*>(p)[i] = w[i];
  }
};

__device__ __forceinline__ void store_codes(uint8_t* p, const float* x, float scale) {
  u32x2 w;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i] / scale, x[4 * i + 1] / scale, 0, false);
    w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2] / scale, x[4 * i + 3] / scale, v, true);
  }
  *reinterpret_cast<u32x2*>(p) = w;
}

struct AppendPlan {
  int32_t lanes, lane_bits;  // of a row
  int32_t tokens;            // of a workgroup
};

template <int DT, bool E4M3>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(const KvAppend a, const AppendPlan p) {
  constexpr int kBytes = value_elem_bytes(DT);
  __shared__ alignas(16) float table[kMaxTable];
  __shared__ alignas(8) uint8_t turned[kMaxTable / 2];
  const int tid = threadIdx.x, dim = a.pages.dim, heads = a.pages.heads, half = a.rot >> 1;
  const int rows = a.q_heads + 2 * heads;
  const int64_t t0 = (int64_t)blockIdx.x * p.tokens;
  const int tokens = (int)min((int64_t)p.tokens, a.tokens - t0);
  const int lane = tid & (p.lanes - 1), turning = a.rot >> 4;  // lanes that rotate
  const int step = kThreads >> p.lane_bits;

  // Where a lane's two times 8 values of a row are; `have`: how many of the two exist.
  struct Place {
    int first, second, have;
    bool turn;
  };
  auto place = [&](bool value) {
    Place r;
    r.turn = !value && lane < turning;
    if (r.turn && !a.interleaved) {
      r.first = 8 * lane;
      r.second = half + 8 * lane;
    } else {
      r.first = 16 * lane;  // the unrotated rest starts at rot = 16 * turning
      r.second = r.first + 8;
    }
    r.have = r.turn ? 2 : r.first + 8 < dim ? 2 : r.first < dim ? 1 : 0;
    return r;
  };
  struct Row {
    int64_t t;
    int head, kind;  // kind: 0 query, 1 key, 2 value
  };
  auto row_at = [&](int r) {
    Row x;
    const int token = r / rows;
    x.t = t0 + token;
    x.head = r - token * rows;
    x.kind = x.head < a.q_heads ? 0 : x.head < a.q_heads + heads ? 1 : 2;
    x.head -= x.kind == 0 ? 0 : x.kind == 1 ? a.q_heads : a.q_heads + heads;
    return x;
  };
  Eight<DT> x0, x1;
  auto load = [&](int r) {
    const Row u = row_at(r);
    const Place at = place(u.kind == 2);
    const KvRows& in = u.kind == 0 ? a.q : u.kind == 1 ? a.k : a.v;
    const uint8_t* row = in.p + (u.t * in.token_stride + u.head * in.head_stride) * kBytes;
    if (at.have > 0) x0.load(row + at.first * kBytes);
    if (at.have > 1) x1.load(row + at.second * kBytes);
  };

  int r = tid >> p.lane_bits;
  const int all = tokens * rows;
  if (r < all) load(r);
  for (int e = tid; e < tokens * a.rot; e += kThreads) {
    const int token = e / a.rot, i = e - token * a.rot, pair = i < half ? i : i - half;
    const int64_t pos = a.positions[axis_of(a, pair) * a.axis_stride + t0 + token];
    const bool in = pos >= 0 && pos < a.max_position;
    table[e] = in ? a.cos_sin[pos * a.rot + i] : 0.0f;
    if (i < half) turned[token * half + i] = in;
  }
  __syncthreads();

  while (r < all) {
    const Row u = row_at(r);
    const Place at = place(u.kind == 2);
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = 0.0f;
    if (at.have > 0) x0.get(x);
    if (at.have > 1) x1.get(x + 8);
    const int next = r + step;
    if (next < all) load(next);
    if (at.turn) {
      // pair i of the lane: values i and i + 8, or 2 i and 2 i + 1
      const f32x4* cos = reinterpret_cast<const f32x4*>(table + (u.t - t0) * a.rot + 8 * lane);
      const f32x4* sin = reinterpret_cast<const f32x4*>(table + (u.t - t0) * a.rot + 8 * lane + half);
      const f32x4 c[2] = {cos[0], cos[1]}, s[2] = {sin[0], sin[1]};
      const uint64_t on = *reinterpret_cast<const uint64_t*>(turned + (u.t - t0) * half + 8 * lane);
      auto turn = [&](float& v, float& w, int i) {
        const float co = c[i / 4][i % 4], si = s[i / 4][i % 4];
        const float y = v * co - w * si, z = w * co + v * si;
        const bool yes = (on >> (8 * i)) & 1;
        v = yes ? y : v;
        w = yes ? z : w;
      };
      if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 8; ++i) turn(x[2 * i], x[2 * i + 1], i);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) turn(x[i], x[8 + i], i);
      }
    }
    if (u.kind == 0) {
      uint8_t* out = a.q_out + (u.t * a.q_out_token_stride + u.head * a.q_out_head_stride) * kBytes;
      if (at.have > 0) Eight<DT>::store(out + at.first * kBytes, x);
      if (at.have > 1) Eight<DT>::store(out + at.second * kBytes, x + 8);
    } else {
      const int64_t to = row_of(a, u.t, u.head);
      uint8_t* pages = u.kind == 2 ? a.pages.v : a.pages.k;
      if constexpr (E4M3) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = max(top, magnitude(x[i]));
        for (int m = p.lanes >> 1; m > 0; m >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m));
        const float scale = e4m3_scale(top);
        if (to >= 0) {
          if (at.have > 0) store_codes(pages + to * dim + at.first, x, scale);
          if (at.have > 1) store_codes(pages + to * dim + at.second, x + 8, scale);
          if (lane == 0) (u.kind == 2 ? a.pages.v_scale : a.pages.k_scale)[to] = scale;
        }
      } else if (to >= 0) {
        uint8_t* out = pages + to * dim * kBytes;
        if (at.have > 0) Eight<DT>::store(out + at.first * kBytes, x);
        if (at.have > 1) Eight<DT>::store(out + at.second * kBytes, x + 8);
      }
      if (u.kind == 2 && lane == 0 && to >= 0) write_slot(a, u.t, to);
    }
    r = next;
  }
}

// ---------------------------------------------------------------------------
// any alignment, any rotated width
// ---------------------------------------------------------------------------
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
  const int64_t p = a.positions[axis_of(a, pair) * a.axis_stride + t];
  if (p < 0 || p >= a.max_position) return x;
  const float* cs = a.cos_sin + p * a.rot;
  const float c = cs[pair], s = cs[pair + half], y = (float)row[other];
  return first ? x * c - y * s : x * c + y * s;
}

template <int DT, bool E4M3>
__global__ __launch_bounds__(64 * kRowsPerBlock) void kv_append_any_kernel(const KvAppend a) {
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
  const int64_t at = row_of(a, t, head);
  if (at < 0) return;
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
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kMaxPer; ++i) top = max(top, magnitude(x[i]));
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m));
    const float scale = e4m3_scale(top);
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
  if (lane == 0 && value) write_slot(a, t, at);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
constexpr int64_t kEnough = 2048;  // workgroups
constexpr int64_t kMostGroups = 0xffffffffu / kThreads;  // a launch has fewer than 2^32 threads
static_assert(kThreads == 64 * kRowsPerBlock);

// The n tokens from t0 on.
KvAppend part(const KvAppend& a, int64_t t0, int64_t n) {
  const int e = value_elem_bytes(a.dtype);
  KvAppend r = a;
  r.tokens = n;
  r.slots += t0;
  for (KvRows* rows : {&r.k, &r.v, &r.q})
    if (rows->p) rows->p += t0 * rows->token_stride * e;
  if (r.q_out) r.q_out += t0 * r.q_out_token_stride * e;
  if (r.index) r.index += t0;
  if (r.positions) r.positions += t0;
  return r;
}

bool wide(const KvAppend& a) {
  const int e = value_elem_bytes(a.dtype);
  auto at16 = [&](const void* p, int64_t token, int64_t head) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && token * e % 16 == 0 && head * e % 16 == 0;
  };
  // rows of an e4m3 cache are written 8 bytes at a time, the others' start at 16 bytes with head_dim
  return a.rot % 16 == 0 && at16(a.k.p, a.k.token_stride, a.k.head_stride) &&
         at16(a.v.p, a.v.token_stride, a.v.head_stride) &&
         (a.q_heads == 0 || (at16(a.q.p, a.q.token_stride, a.q.head_stride) &&
                             at16(a.q_out, a.q_out_token_stride, a.q_out_head_stride)));
}

template <int DT, bool E4M3>
hipError_t launch(const KvAppend& a, hipStream_t stream) {
  const int rows = a.q_heads + 2 * a.pages.heads;
  AppendPlan p{};
  int64_t most;  // tokens of a launch
  const bool in_words = wide(a);
  if (in_words) {
    const int need = (a.pages.dim + 15) / 16;
    while ((1 << p.lane_bits) < need) ++p.lane_bits;
    p.lanes = 1 << p.lane_bits;
    // whole tokens: enough to fill the workgroup's threads, and more once there are workgroups for every CU
    const int64_t fill = std::max(1, kThreads / (rows * p.lanes));
    p.tokens = (int)std::max(fill, std::min<int64_t>(8 * fill, a.tokens / kEnough));
    if (a.rot > 0) p.tokens = std::min(p.tokens, kMaxTable / a.rot);
    most = kMostGroups * p.tokens;
  } else {
    most = kMostGroups * kRowsPerBlock / rows;
  }
  for (int64_t t0 = 0; t0 < a.tokens; t0 += most) {
    const KvAppend b = part(a, t0, std::min(most, a.tokens - t0));
    if (in_words)
      kv_append_kernel<DT, E4M3><<<(unsigned)((b.tokens + p.tokens - 1) / p.tokens), kThreads, 0, stream>>>(b, p);
    else
      kv_append_any_kernel<DT, E4M3>
          <<<(unsigned)((b.tokens * rows + kRowsPerBlock - 1) / kRowsPerBlock), kThreads, 0, stream>>>(b);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace

hipError_t launch_kv_append(const KvAppend& a, hipStream_t stream) {
  if (a.tokens == 0) return hipSuccess;
  const bool q8 = a.pages.dtype == kE4M3;
  switch (a.dtype) {
    case kF32: return launch<kF32, false>(a, stream);
    case kF16: return q8 ? launch<kF16, true>(a, stream) : launch<kF16, false>(a, stream);
    case kBF16: return q8 ? launch<kBF16, true>(a, stream) : launch<kBF16, false>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace nve_amd
