// kv_append.hip -- new tokens enter the paged key-value cache: norms of query and key
// heads, rotary positions on them, keys and values written to their slots.
//
// Every value is read and written once, with 3 flops a rotated value and 3 more under a
// norm: bound by the bytes.  kv_append_kernel: a head row is a group of lanes (a power of
// two), 16 values a lane.  A lane that rotates has 8 pairs, both values of each, so
// that nothing crosses lanes but a norm's sum and a scaled row's largest magnitudes: values
// 8 j .. and rot / 2 + 8 j .. of the row, or (pairs of neighbours) 16 j ..; the lanes
// behind them have 16 unrotated values.  A workgroup has whole tokens: it brings
// their cosines and sines into shared memory once for all their heads, while the
// first rows' loads are under way.
// Measured: 16,001 f16 tokens of 32 query and 8 key heads of 128 values 83 us (4.8 TB/s; a
// large copy 4.7 to 5.0); 12,001 of them with norms 63 us (4.8 TB/s); 9,000 bf16 tokens of 96 values
// into e4m3 40 us (3.9 TB/s; 6 of 8 lanes a row work), of 128 values with norms into 4 bits 43 us
// (4.5 TB/s); a step of 64 tokens 4.8 us, with norms 5.7: the chain position, cosine, shared memory, store.
// kv_append_any_kernel, for rows that start off 16 bytes and for rotated widths
// that are no multiple of 16 (4-bit pages, pairs of halves: of 64, so that 32 values of a scale
// are in neighbouring lanes): one value of a row per lane and step (409 us for the
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

// The exponent byte of the scale of 32 kMXFP4 values whose largest magnitude has the bits `top`:
// the least power of two with top <= 7 times it, so that no value is further from a multiple than
// half the widest step (4 to 6).  top is 1.75 * 4 times a power of two at most where its fraction is
// 0x600000 at most, hence the carry.
__device__ __forceinline__ uint32_t mxfp4_exponent(uint32_t top) {
  return top >= 0x7f800000u ? 255u : max((top + 0x1fffffu) >> 23, 3u) - 2u;
}
__device__ __forceinline__ float mxfp4_scale(uint32_t exponent) { return __uint_as_float(exponent << 23); }

// 8 values' codes, the first one's lowest.
__device__ __forceinline__ uint32_t mxfp4_codes(const float* x, float scale) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
  return w;
}

// 1 / sqrt(mean square + eps) of a row whose squares' sum is `sum`.  The sum is in 64 bits: what
// follows is f32 steps that any order of it leaves alike, and 4- and 8-bit codes do not turn on it.
// The instruction's root (some 2^-26 off) and the next two terms of its error's series, in place of a
// root and two divisions: 12,001 f16 tokens of 32 query and 8 key heads 81 -> 68 us.
__device__ __forceinline__ float inverse_rms(double sum, double inverse_dim, double eps) {
  const double y = fma(sum, inverse_dim, eps), r = __builtin_amdgcn_rsq(y);
  const double e = fma(-(y * r), r, 1.0);
  // 0 and infinity have no e, and their root as it is
  return (float)(e == e ? fma(r * e, fma(e, 0.375, 0.5), r) : r);
}

// The sum over a row's lanes, 2^bits neighbours.
template <int CTRL>
__device__ __forceinline__ double of_neighbour(double x) {
  uint32_t w[2];
  __builtin_memcpy(w, &x, 8);
#pragma unroll
  for (int i = 0; i < 2; ++i) w[i] = (uint32_t)__builtin_amdgcn_mov_dpp((int)w[i], CTRL, 0xf, 0xf, false);
  __builtin_memcpy(&x, w, 8);
  return x;
}
__device__ __forceinline__ double lanes_sum(double x, int bits) {
  if (bits >= 1) x += of_neighbour<0xb1>(x);   // the lane beside
  if (bits >= 2) x += of_neighbour<0x4e>(x);   // the pair beside
  if (bits >= 3) x += of_neighbour<0x141>(x);  // the four beside: half a row of 16 mirrored
  if (bits >= 4) x += of_neighbour<0x140>(x);  // a row mirrored
  return x;
}

struct AppendPlan {
  int32_t lanes, lane_bits;  // of a row
  int32_t tokens;            // of a workgroup
};

// DT: the rows' type, CT: the pages'; NORM: queries or keys have a norm.
template <int DT, int CT, bool NORM>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(const KvAppend a, const AppendPlan p) {
  constexpr int kBytes = value_elem_bytes(DT);
  __shared__ alignas(16) float table[kMaxTable];
  __shared__ alignas(8) uint8_t turned[kMaxTable / 2];
  __shared__ alignas(16) float norms[NORM ? 2 : 1][NORM ? 256 : 4];  // of queries and of keys
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
  if constexpr (NORM) {
    using T = kv_elem<DT>;
    norms[0][tid] = a.q_norm && tid < dim ? (float)reinterpret_cast<const T*>(a.q_norm)[tid] : 0.0f;
    norms[1][tid] = a.k_norm && tid < dim ? (float)reinterpret_cast<const T*>(a.k_norm)[tid] : 0.0f;
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
    if constexpr (NORM) {
      if (u.kind == 0 ? a.q_norm != nullptr : u.kind == 1 && a.k_norm != nullptr) {
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < 16; ++i) sum = fma((double)x[i], (double)x[i], sum);
        const float f = inverse_rms(lanes_sum(sum, p.lane_bits), a.inverse_dim, a.eps);
        const f32x4* w0 = reinterpret_cast<const f32x4*>(&norms[u.kind][at.first]);
        const f32x4* w1 = reinterpret_cast<const f32x4*>(&norms[u.kind][at.second]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = x[i] * f * w0[i / 4][i % 4];
          x[8 + i] = x[8 + i] * f * w1[i / 4][i % 4];
        }
      }
    }
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
      if constexpr (CT == kMXFP4) {
        // 32 values that share a scale: 4 lanes' 8 (two such runs), or 2 lanes' 16
        uint32_t top[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 16; ++i) top[i / 8] = max(top[i / 8], magnitude(x[i]));
        const bool apart = at.turn && !a.interleaved;
        if (!apart) top[0] = top[1] = max(top[0], top[1]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          top[i] = max(top[i], (uint32_t)__shfl_xor((int)top[i], 1));
          if (apart) top[i] = max(top[i], (uint32_t)__shfl_xor((int)top[i], 2));
        }
        if (to >= 0 && at.have > 0) {  // dim is a multiple of 32: both halves are there
          uint8_t* codes = pages + to * (dim / 2);
          uint8_t* scales = static_cast<uint8_t*>(u.kind == 2 ? a.pages.v_scale : a.pages.k_scale) + to * (dim / 32);
          const int first[2] = {at.first, at.second};
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t e = mxfp4_exponent(top[i]);
            *reinterpret_cast<uint32_t*>(codes + first[i] / 2) = mxfp4_codes(x + 8 * i, mxfp4_scale(e));
            if (first[i] % 32 == 0) scales[first[i] / 32] = (uint8_t)e;
          }
        }
      } else if constexpr (CT == kE4M3) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = max(top, magnitude(x[i]));
        for (int m = p.lanes >> 1; m > 0; m >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m));
        const float scale = e4m3_scale(top);
        if (to >= 0) {
          if (at.have > 0) store_codes(pages + to * dim + at.first, x, scale);
          if (at.have > 1) store_codes(pages + to * dim + at.second, x + 8, scale);
          if (lane == 0) static_cast<float*>(u.kind == 2 ? a.pages.v_scale : a.pages.k_scale)[to] = scale;
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

// A row's norm: every value times f and its weight (null: no norm).
template <typename T>
struct Norm {
  const T* weight;
  float f;
  __device__ __forceinline__ float of(const T* row, int d) const {
    const float x = (float)row[d];
    return weight ? x * f * (float)weight[d] : x;
  }
};

// Of a whole wave's row.
template <typename T>
__device__ __forceinline__ Norm<T> norm_of(const KvAppend& a, const uint8_t* weight, const T* row, int lane) {
  Norm<T> n{reinterpret_cast<const T*>(weight), 1.0f};
  if (!weight) return n;
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < kMaxPer; ++i) {
    const int d = lane + 64 * i;
    const double x = d < a.pages.dim ? (double)(float)row[d] : 0.0;
    sum = fma(x, x, sum);
  }
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) sum += __shfl_xor(sum, m);
  n.f = inverse_rms(sum, a.inverse_dim, a.eps);
  return n;
}

// Value d of a head row of token t, normed and rotated; f32 products and sum rounded one by one.
template <typename T>
__device__ __forceinline__ float rotated(const KvAppend& a, const Norm<T>& norm, const T* row, int64_t t, int d) {
  const float x = norm.of(row, d);
  if (d >= a.rot) return x;
  const int half = a.rot >> 1;
  const int pair = a.interleaved ? d >> 1 : (d < half ? d : d - half);
  const bool first = a.interleaved ? (d & 1) == 0 : d < half;
  const int other = a.interleaved ? d ^ 1 : (first ? d + half : d - half);
  const int64_t p = a.positions[axis_of(a, pair) * a.axis_stride + t];
  if (p < 0 || p >= a.max_position) return x;
  const float* cs = a.cos_sin + p * a.rot;
  const float c = cs[pair], s = cs[pair + half], y = norm.of(row, other);
  return first ? x * c - y * s : x * c + y * s;
}

template <int DT, int CT>
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
    const Norm<T> norm = norm_of(a, a.q_norm, row, lane);
    float x[kMaxPer];
#pragma unroll
    for (int i = 0; i < kMaxPer; ++i)
      if (lane + 64 * i < dim) x[i] = rotated(a, norm, row, t, lane + 64 * i);
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
  const Norm<T> norm = norm_of(a, value ? nullptr : a.k_norm, row, lane);
  float x[kMaxPer];
#pragma unroll
  for (int i = 0; i < kMaxPer; ++i) {
    const int d = lane + 64 * i;
    x[i] = d >= dim ? 0.0f : value ? (float)row[d] : rotated(a, norm, row, t, d);
  }
  if constexpr (CT == kMXFP4) {
    uint8_t* scales = static_cast<uint8_t*>(value ? a.pages.v_scale : a.pages.k_scale) + at * (dim / 32);
#pragma unroll
    for (int i = 0; i < kMaxPer; ++i) {  // half a wave has 32 values of a scale, or none
      const int d = lane + 64 * i;
      uint32_t top = magnitude(x[i]);
#pragma unroll
      for (int m = 16; m > 0; m >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m));
      const uint32_t e = mxfp4_exponent(top);
      const float next = __shfl_xor(x[i], 1);
      const uint32_t codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, x[i], next, mxfp4_scale(e), 0);
      if (d < dim && lane % 2 == 0) pages[at * (dim / 2) + d / 2] = (uint8_t)codes;
      if (d < dim && d % 32 == 0) scales[d / 32] = (uint8_t)e;
    }
  } else if constexpr (CT == kE4M3) {
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
    if (lane == 0) static_cast<float*>(value ? a.pages.v_scale : a.pages.k_scale)[at] = scale;
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
constexpr int64_t kEnough = 640;  // workgroups
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
  // rows of an e4m3 cache are written 8 bytes at a time, the others' start at 16 bytes with head_dim;
  // 32 values with a scale of their own have to be in 4 lanes, or in 2 with 16 each
  return a.rot % (a.pages.dtype == kMXFP4 && !a.interleaved ? 64 : 16) == 0 && at16(a.k.p, a.k.token_stride, a.k.head_stride) &&
         at16(a.v.p, a.v.token_stride, a.v.head_stride) &&
         (a.q_heads == 0 || (at16(a.q.p, a.q.token_stride, a.q.head_stride) &&
                             at16(a.q_out, a.q_out_token_stride, a.q_out_head_stride)));
}

template <int DT, int CT>
hipError_t launch(const KvAppend& a, hipStream_t stream) {
  const int rows = a.q_heads + 2 * a.pages.heads;
  AppendPlan p{};
  int64_t most;  // tokens of a launch
  const bool in_words = wide(a), norm = a.q_norm || a.k_norm;
  if (in_words) {
    const int need = (a.pages.dim + 15) / 16;
    while ((1 << p.lane_bits) < need) ++p.lane_bits;
    p.lanes = 1 << p.lane_bits;
    // Whole tokens: enough to fill the workgroup's threads, and more, while there are workgroups for every CU, where
    // their rows leave fewer threads idle in the last turn (12,001 tokens of 48 rows of 8 lanes: 1 token 77.5 us, 2
    // 63.5, 5 67.3; 4,801 of 36 rows of 4 lanes, 64 f32 values: 1 26.2, 2 26.9, 5 24.5, 7 23.8).
    const int64_t each = (int64_t)rows * p.lanes, fill = std::max<int64_t>(1, kThreads / each);
    int64_t most_tokens = std::max(fill, std::min(8 * fill, a.tokens / kEnough));
    if (a.rot > 0) most_tokens = std::min<int64_t>(most_tokens, kMaxTable / a.rot);
    auto busy = [&](int64_t tokens) { return (double)(tokens * each) / ((tokens * each + kThreads - 1) / kThreads * kThreads); };
    p.tokens = (int)std::min(fill, most_tokens);
    for (int64_t t = p.tokens + 1; t <= most_tokens; ++t)
      if (busy(t) > busy(p.tokens) + 0.03) p.tokens = (int)t;
    most = kMostGroups * p.tokens;
  } else {
    most = kMostGroups * kRowsPerBlock / rows;
  }
  for (int64_t t0 = 0; t0 < a.tokens; t0 += most) {
    const KvAppend b = part(a, t0, std::min(most, a.tokens - t0));
    const unsigned groups = in_words ? (unsigned)((b.tokens + p.tokens - 1) / p.tokens) : 0;
    if (in_words && norm)
      kv_append_kernel<DT, CT, true><<<groups, kThreads, 0, stream>>>(b, p);
    else if (in_words)
      kv_append_kernel<DT, CT, false><<<groups, kThreads, 0, stream>>>(b, p);
    else
      kv_append_any_kernel<DT, CT>
          <<<(unsigned)((b.tokens * rows + kRowsPerBlock - 1) / kRowsPerBlock), kThreads, 0, stream>>>(b);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <int DT>
hipError_t launch_pages(const KvAppend& a, hipStream_t stream) {
  switch (a.pages.dtype) {
    case kE4M3: return launch<DT, kE4M3>(a, stream);
    case kMXFP4: return launch<DT, kMXFP4>(a, stream);
    default: return launch<DT, DT>(a, stream);
  }
}

}  // namespace

hipError_t launch_kv_append(const KvAppend& a, hipStream_t stream) {
  if (a.tokens == 0) return hipSuccess;
  switch (a.dtype) {
    case kF32: return launch<kF32, kF32>(a, stream);
    case kF16: return launch_pages<kF16>(a, stream);
    case kBF16: return launch_pages<kBF16>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace nve_amd
