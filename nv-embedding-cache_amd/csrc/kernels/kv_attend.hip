// kv_attend.hip -- attention of one new token per sequence over its pages.
//
// For a query head h and the slots t of its sequence: x_t = scale q . k_t,
// p = softmax(x), out = sum p_t v_t.  One pass over k and v with the running
// maximum m and sum l of the softmax; what was summed before is scaled by
// 2^(m_old - m) when the maximum grows (x in units of log2).
//
// Bound: every k and v row is read once for 4 flops per query head and byte
// pair, so the pages' bytes bound it; the matrix instructions keep the work per
// byte far below that, whatever the group of query heads (up to 16) that
// shares a key head.
//
// Layout of a wave's step (kStep slots, 16 query columns).  Scores are computed
// transposed: S^T = K Q^T, the k rows as the A operand (a lane reads 16 bytes of
// one row at a time, as they lie in the page) and the queries as B, kept in
// registers.  Then a lane holds, for one query (lane % 16), the scores of 4
// slots per tile of 16 (4 (lane / 16) ..), and the weights it makes of them are
// already the B operand of out^T = V^T P^T: nothing crosses lanes but the
// maximum.  The A operand V^T wants one value of 8 slots per lane: a lane reads
// the same piece of its 8 slots' rows and transposes 16-bit pairs in registers.
// A value tile's row r is the value r * dim / 16 + tile, which makes those
// pieces contiguous.  No shared memory until the waves of a workgroup join.
//
// Weights enter the second product as the sum of two values of the product's
// type (at least 16 bits of the f32 weight): one alone would lose as much as the
// output's own rounding, and the matrix units are idle anyway.  f16 weights are
// held times 2^14, so that a long flat tail does not underflow (2^-38 of the
// maximum still counts).  e4m3 rows are widened exactly to the query's type
// (scores) and to bf16 (values); their scales go into scores and weights.
//
// Split: workgroups of 4 waves are the machine's resident ones, and each takes
// an equal run of the tiles (4 kStep slots) of all (sequence, key head, 16
// queries) units laid end to end, whatever the lengths.  A unit inside one
// workgroup is finished there; pieces of a unit go to the workspace as f32 rows
// with their m and l, and the second kernel, mapped the same way, joins them.
// It also adds the attention weights where they are asked for, from the scores
// that the first kernel left in the workspace.
#include <math.h>

#include <algorithm>

#include <type_traits>

#include "kv_common.cuh"

namespace nve_amd {

namespace {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// f32 has 4 slots per lane and step, the other types 8.
constexpr int step_slots(int qt) { return qt == kF32 ? 16 : 32; }
constexpr int tile_slots(int qt) { return kWaves * step_slots(qt); }

// ---------------------------------------------------------------------------
// the workgroups' shares
// ---------------------------------------------------------------------------
struct Plan {
  int64_t units_per_seq;  // key heads * query tiles
  int32_t query_tiles, group, tile;
  int64_t padded;   // slots of a row of scores
  float* scores;    // [seqs * q_heads, padded], log2 units (accumulate)
  float* sums;      // [units, 16]: log2 of the softmax's sum (accumulate)
  float* slot_ml;   // [2 * workgroups, 2, 16]
  float* slot_rows; // [2 * workgroups, 16, dim padded]
};

// Tiles of a sequence; one at least, so that an empty one is visited.
__device__ __forceinline__ int64_t tiles_of(const KvAttend& a, const Plan& p, int64_t s) {
  const int64_t n = kv_length(a.lengths, s, a.max_length);
  return n <= p.tile ? 1 : (n + p.tile - 1) / p.tile;
}

struct Share {
  int64_t total;         // tiles of the call
  int64_t workers;       // workgroups that have a share: no share is empty
  int64_t begin, end;    // this workgroup's
  int64_t seq, seq_tile; // the sequence `begin` lies in, and the call's tile where it starts
};

__device__ __forceinline__ int64_t share_begin(const Share& s, int64_t w) { return w * s.total / s.workers; }
// the workgroup that has a tile
__device__ __forceinline__ int64_t share_of(const Share& s, int64_t tile) {
  return ((tile + 1) * s.workers - 1) / s.total;
}

// Every thread sums a run of the sequences; a scan finds where the share starts.
__device__ __forceinline__ Share find_share(const KvAttend& a, const Plan& p) {
  __shared__ int64_t wave_total[kWaves];
  __shared__ int64_t found[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t per = (a.seqs + kThreads - 1) / kThreads;
  const int64_t s0 = per * tid < a.seqs ? per * tid : a.seqs;
  const int64_t s1 = s0 + per < a.seqs ? s0 + per : a.seqs;
  int64_t own = 0;
  for (int64_t s = s0; s < s1; ++s) own += tiles_of(a, p, s);
  int64_t scan = own;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t o = __shfl_up(scan, d);
    if (lane >= d) scan += o;
  }
  if (lane == 63) wave_total[wave] = scan;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) scan += wave_total[w];
    total += wave_total[w];
  }
  Share r;
  r.total = total * p.units_per_seq;
  r.workers = r.total < gridDim.x ? r.total : gridDim.x;
  if (blockIdx.x >= r.workers) {
    r.begin = r.end = r.total;
    return r;
  }
  r.begin = share_begin(r, blockIdx.x);
  r.end = share_begin(r, (int64_t)blockIdx.x + 1);
  int64_t at = (scan - own) * p.units_per_seq;
  if (r.begin >= at && r.begin < scan * p.units_per_seq) {
    int64_t s = s0;
    for (; s < s1; ++s) {
      const int64_t n = tiles_of(a, p, s) * p.units_per_seq;
      if (r.begin < at + n) break;
      at += n;
    }
    found[0] = s;
    found[1] = at;
  }
  __syncthreads();
  r.seq = found[0];
  r.seq_tile = found[1];
  return r;
}

// A run of one unit's tiles in a workgroup's share.
struct Piece {
  int64_t seq, len, tiles;  // the unit's
  int64_t unit_tile;        // the call's tile where the unit starts
  int64_t first, last;      // [first, last) of the unit's tiles
  int64_t unit;
  int head, query_tile;
};

__device__ __forceinline__ Piece piece_at(const KvAttend& a, const Plan& p, int64_t tile, int64_t end, int64_t seq,
                                          int64_t seq_tile) {
  Piece r;
  r.seq = seq;
  r.len = kv_length(a.lengths, seq, a.max_length);
  r.tiles = r.len <= p.tile ? 1 : (r.len + p.tile - 1) / p.tile;
  const int64_t u = (tile - seq_tile) / r.tiles;
  r.unit = seq * p.units_per_seq + u;
  r.head = (int)(u / p.query_tiles);
  r.query_tile = (int)(u - (int64_t)r.head * p.query_tiles);
  r.unit_tile = seq_tile + u * r.tiles;
  r.first = tile - r.unit_tile;
  r.last = end - r.unit_tile < r.tiles ? end - r.unit_tile : r.tiles;
  return r;
}

// ---------------------------------------------------------------------------
// lane helpers
// ---------------------------------------------------------------------------
// Maximum and sum over the four lanes that hold one query (lane % 16).
__device__ __forceinline__ float query_max(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float query_sum(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// v_exp_f32: 2^-infinity is 0; results below the normal range flush to 0.
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// 2^(m - base) where m may be -infinity (a maximum over nothing).
__device__ __forceinline__ float rescale(float m, float base) { return m == -INFINITY ? 0.0f : exp2_of(m - base); }

template <int QT>
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (QT == kF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
}

template <int QT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (QT == kF16) {
    using half2 = __attribute__((ext_vector_type(2))) _Float16;
    return __builtin_bit_cast(uint32_t, half2{(_Float16)a, (_Float16)b});
  } else {
    using bhalf2 = __attribute__((ext_vector_type(2))) __bf16;
    return __builtin_bit_cast(uint32_t, bhalf2{(__bf16)a, (__bf16)b});
  }
}
template <int QT>
__device__ __forceinline__ float low_of(uint32_t w) {
  if constexpr (QT == kF16) return (float)__builtin_bit_cast(_Float16, (uint16_t)w);
  else return __uint_as_float(w << 16);
}
template <int QT>
__device__ __forceinline__ float high_of(uint32_t w) {
  if constexpr (QT == kF16) return (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16));
  else return __uint_as_float(w & 0xffff0000u);
}

// Two e4m3 codes (the low or high half of w) widened exactly.
template <int QT, bool HIGH>
__device__ __forceinline__ uint32_t widen2(uint32_t w) {
  const auto x = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, HIGH);
  return pack2<QT>(x[0], x[1]);
}

// 8 or 16 bytes of a row (any 4-byte alignment).
template <int WORDS>
__device__ __forceinline__ void load_words(uint32_t* dst, const uint8_t* src) {
  using gwords = const __attribute__((address_space(1))) uint32_t*;
  gwords p = (gwords)(uintptr_t)src;
  if constexpr (WORDS == 4) {
    typedef u32x4 __attribute__((aligned(4))) u4;
    const u32x4 x = *(const __attribute__((address_space(1))) u4*)p;
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[i] = x[i];
  } else if constexpr (WORDS == 2) {
    typedef uint64_t __attribute__((aligned(4))) u2;
    const uint64_t x = *(const __attribute__((address_space(1))) u2*)p;
    dst[0] = (uint32_t)x;
    dst[1] = (uint32_t)(x >> 32);
  } else {
    dst[0] = *p;
  }
}

// ---------------------------------------------------------------------------
// the first kernel
// ---------------------------------------------------------------------------
// DP: head_dim rounded up to 64, 128 or 256; EXACT: head_dim is DP.
template <int QT, int CT, int DP, bool EXACT>
struct Wave {
  static constexpr int kStep = step_slots(QT);
  static constexpr int kTiles = kStep / 16;        // score tiles of a step
  static constexpr int kSlots = kStep / 4;         // slots of a lane
  static constexpr int kBytes = value_elem_bytes(CT);
  static constexpr int kPieces = DP * kBytes / 64; // 16-byte pieces of a k row in a lane
  static constexpr int kSteps = DP / 32;           // 16-bit products of a row
  static constexpr int kValues = DP / 16;          // values of a v row in a lane, and output tiles
  static constexpr int kVWords = kValues * kBytes / 4;
  static constexpr int VT = CT == kE4M3 ? kBF16 : QT;  // the type of the second product
  static constexpr int kQWords = QT == kF32 ? DP / 4 : kSteps * 4;

  uint32_t q[kQWords];
  uint32_t k[kTiles][kPieces * 4];
  uint32_t v[kSlots][kVWords];
  f32x4 acc[kValues];
  float m, l;  // m: of the query; l: of this lane's slots

  // The value of a row where word w of a lane's queries starts.
  static __device__ __forceinline__ int q_value(int w, int g) {
    if constexpr (QT == kF32) return (w >> 2) * 16 + g * 4 + (w & 3);
    const int step = w >> 2, i = (w & 3) * 2;
    if constexpr (CT == kE4M3) return (step >> 1) * 64 + g * 16 + (step & 1) * 8 + i;
    return step * 32 + g * 8 + i;
  }

  __device__ __forceinline__ void load_queries(const KvAttend& a, int64_t row_offset, bool there, int g) {
    const int dim = a.pages.dim;
#pragma unroll
    for (int w = 0; w < kQWords; ++w) {
      const int d = q_value(w, g);
      q[w] = 0;
      if (!there || (!EXACT && d >= dim)) continue;
      if constexpr (QT == kF32) {
        q[w] = reinterpret_cast<const uint32_t*>(a.q.p)[row_offset + d];
      } else {
        const uint16_t* p = reinterpret_cast<const uint16_t*>(a.q.p) + row_offset + d;
        q[w] = p[0] | (uint32_t)p[1] << 16;
      }
    }
  }

  // A k row's pieces: 16 bytes at 64 i + 16 g.
  static __device__ __forceinline__ void load_k(uint32_t (&r)[kPieces * 4], const uint8_t* row, int g, int dim) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int b = i * 64 + g * 16;
      if constexpr (EXACT) {
        load_words<4>(&r[4 * i], row + b);
      } else if constexpr (CT == kE4M3) {  // head_dim is a multiple of 8: half a piece
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          r[4 * i + 2 * h] = r[4 * i + 2 * h + 1] = 0;
          if (b + 8 * h < dim) load_words<2>(&r[4 * i + 2 * h], row + b + 8 * h);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) r[4 * i + j] = 0;
        if (b < dim * kBytes) load_words<4>(&r[4 * i], row + b);
      }
    }
  }

  // A v row's values kValues c ..; those past head_dim are not used (the row's first instead).
  static __device__ __forceinline__ void load_v(uint32_t (&r)[kVWords], const uint8_t* row, int c, int dim) {
    const int b = c * kValues * kBytes;
    constexpr int kLoad = EXACT ? (kVWords < 4 ? kVWords : 4) : CT == kE4M3 ? (kVWords < 2 ? 1 : 2) : (kVWords < 4 ? kVWords : 4);
#pragma unroll
    for (int i = 0; i < kVWords; i += kLoad) {
      const int at = b + 4 * i;
      load_words<kLoad>(&r[i], row + (EXACT || at < dim * kBytes ? at : 0));
    }
  }

  __device__ __forceinline__ f32x4 scores(int tile) const {
    f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (QT == kF32) {
#pragma unroll
      for (int w = 0; w < DP / 4; ++w)
        s = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[tile][w]), __uint_as_float(q[w]), s, 0, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const u32x4 b = {q[4 * i], q[4 * i + 1], q[4 * i + 2], q[4 * i + 3]};
        u32x4 x;
        if constexpr (CT == kE4M3) {
          const uint32_t w0 = k[tile][2 * i], w1 = k[tile][2 * i + 1];
          x = u32x4{widen2<QT, false>(w0), widen2<QT, true>(w0), widen2<QT, false>(w1), widen2<QT, true>(w1)};
        } else {
          x = u32x4{k[tile][4 * i], k[tile][4 * i + 1], k[tile][4 * i + 2], k[tile][4 * i + 3]};
        }
        s = mma<QT>(x, b, s);
      }
    }
    return s;
  }

  // acc += V^T P^T for the weights p of this lane's slots.
  __device__ __forceinline__ void add_values(const float (&p)[kSlots]) {
    if constexpr (QT == kF32) {
#pragma unroll
      for (int j = 0; j < kValues; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[r][j]), p[r], acc[j], 0, 0, 0);
    } else {
      u32x4 high, low;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        high[i] = pack2<VT>(p[2 * i], p[2 * i + 1]);
        low[i] = pack2<VT>(p[2 * i] - low_of<VT>(high[i]), p[2 * i + 1] - high_of<VT>(high[i]));
      }
      uint32_t w[8][kValues / 2];
#pragma unroll
      for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int i = 0; i < kValues / 2; ++i) {
          if constexpr (CT == kE4M3)
            w[r][i] = (i & 1) ? widen2<VT, true>(v[r][i / 2]) : widen2<VT, false>(v[r][i / 2]);
          else
            w[r][i] = v[r][i];
        }
#pragma unroll
      for (int j = 0; j < kValues; ++j) {
        u32x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[i] = __builtin_amdgcn_perm(w[2 * i + 1][j / 2], w[2 * i][j / 2], (j & 1) ? 0x07060302u : 0x05040100u);
        acc[j] = mma<VT>(x, high, acc[j]);
        acc[j] = mma<VT>(x, low, acc[j]);
      }
    }
  }
};

template <int QT, int CT, int DP, bool EXACT, bool ACC>
__global__ __launch_bounds__(kThreads) void kv_attend_kernel(const KvAttend a, const Plan p) {
  using W = Wave<QT, CT, DP, EXACT>;
  using T = kv_elem<QT>;
  constexpr int kStep = W::kStep, kValues = W::kValues;
  constexpr int kPass = kValues < 8 ? kValues : 8;  // output tiles joined at a time
  constexpr int kRow = 16 * kPass + 4;              // a query's values in shared memory, padded
  __shared__ float wave_ml[kWaves][2][16];
  __shared__ float rows[kWaves][16 * kRow];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, g = lane >> 4;
  const KvPages& pages = a.pages;
  const int dim = EXACT ? DP : pages.dim;
  const int row_bytes = dim * W::kBytes, mask = pages.page - 1;
  const uint64_t page_bytes = (uint64_t)pages.heads * pages.page * row_bytes;
  const float to_log2 = a.scale * kLog2e;
  const Share share = find_share(a, p);
  int64_t seq = share.seq, seq_tile = share.seq_tile;
  W x;

  for (int64_t tile = share.begin; tile < share.end;) {
    const Piece u = piece_at(a, p, tile, share.end, seq, seq_tile);
    const int rows_here = min(16, p.group - u.query_tile * 16);
    const int64_t q_head = (int64_t)u.head * p.group + u.query_tile * 16 + c;
    const bool there = c < rows_here;
    x.load_queries(a, u.seq * a.q.token_stride + q_head * a.q.head_stride, there, g);
#pragma unroll
    for (int j = 0; j < kValues; ++j) x.acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    x.m = -INFINITY;
    x.l = 0.0f;

    const int32_t* table = a.tables + u.seq * a.table_stride;
    const int steps = (int)(u.last - u.first);
    const int64_t t_base = u.first * (kWaves * kStep) + wave * kStep;  // this wave's first slot
    // Page numbers of 16 steps: lane 4 i + b has that of slots 8 b .. of step i (-1: absent).
    int ids = -1;
    auto load_ids = [&](int step) {
      const int64_t t = t_base + (int64_t)(step + (lane >> 2)) * (kWaves * kStep) + (lane & 3) * 8;
      ids = -1;
      if (t < u.len && (lane & 3) * 8 < kStep) {
        const int64_t id = table[t >> pages.page_bits];
        if (id >= 0 && id < pages.num_pages) ids = (int)id;
      }
    };
    auto row_at = [&](const uint8_t* base, int id, int64_t t) {
      const uint32_t in_page = (uint32_t)(u.head * pages.page + ((int)t & mask)) * (uint32_t)row_bytes;
      return base + (uint64_t)(uint32_t)max(id, 0) * page_bytes + in_page;
    };
    // Slots without a row read the first page's instead; their scores and values are dropped below.
    auto load_k = [&](int step) {
      const int64_t t0 = t_base + (int64_t)step * (kWaves * kStep);
#pragma unroll
      for (int n = 0; n < W::kTiles; ++n) {
        const int id = __shfl(ids, (step & 15) * 4 + n * 2 + (c >> 3));
        W::load_k(x.k[n], row_at(pages.k, id, t0 + n * 16 + c), g, dim);
      }
    };
    auto load_v = [&](int step) {
      const int64_t t0 = t_base + (int64_t)step * (kWaves * kStep);
#pragma unroll
      for (int n = 0; n < W::kTiles; ++n) {
        const int id = __shfl(ids, (step & 15) * 4 + n * 2 + (g >> 1));
        const uint8_t* row = row_at(pages.v, id, t0 + n * 16 + g * 4);
#pragma unroll
        for (int r = 0; r < 4; ++r) W::load_v(x.v[n * 4 + r], row + r * row_bytes, c, dim);
      }
    };

    load_ids(0);
    load_k(0);
    load_v(0);
    for (int step = 0; step < steps; ++step) {
      const int64_t t0 = t_base + (int64_t)step * (kWaves * kStep);
      f32x4 s[W::kTiles];
#pragma unroll
      for (int n = 0; n < W::kTiles; ++n) s[n] = x.scores(n);
      // the four page numbers of this step, -1 where a slot has no row
      const uint64_t absent = __ballot(ids < 0) >> ((step & 15) * 4);
      const bool full = t0 + kStep <= u.len && (absent & (kStep == 32 ? 15 : 3)) == 0;
      float scale_v[W::kSlots];
      float y[W::kSlots];
#pragma unroll
      for (int n = 0; n < W::kTiles; ++n) {
        const int id = __shfl(ids, (step & 15) * 4 + n * 2 + (g >> 1));
        const int64_t t = t0 + n * 16 + g * 4;
        f32x4 ks = {1.0f, 1.0f, 1.0f, 1.0f}, vs = ks;
        if constexpr (CT == kE4M3) {
          const int64_t at = ((int64_t)max(id, 0) * pages.heads + u.head) * pages.page + (t & mask);
          typedef f32x4 __attribute__((aligned(4))) f4;
          ks = *reinterpret_cast<const f4*>(pages.k_scale + at);
          vs = *reinterpret_cast<const f4*>(pages.v_scale + at);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          y[n * 4 + r] = s[n][r] * to_log2;
          scale_v[n * 4 + r] = 1.0f;
          if constexpr (CT == kE4M3) {
            y[n * 4 + r] *= ks[r];
            scale_v[n * 4 + r] = vs[r];
          }
        }
        if (!full) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (id < 0 || t + r >= u.len) {
              y[n * 4 + r] = -INFINITY;
              scale_v[n * 4 + r] = 0.0f;
#pragma unroll
              for (int w = 0; w < W::kVWords; ++w) x.v[n * 4 + r][w] = 0;
            }
        }
        if constexpr (ACC) {
          if (there && t < u.len)  // rows of scores are padded to whole tiles
            *reinterpret_cast<f32x4*>(p.scores + (u.seq * a.q_heads + q_head) * p.padded + t) =
                f32x4{y[n * 4], y[n * 4 + 1], y[n * 4 + 2], y[n * 4 + 3]};
        }
      }
      const bool more = step + 1 < steps;
      if (more && ((step + 1) & 15) == 0) load_ids(step + 1);
      if (more) load_k(step + 1);

      float top = y[0];
#pragma unroll
      for (int i = 1; i < W::kSlots; ++i) top = fmaxf(top, y[i]);
      top = fmaxf(x.m, query_max(top));
      if (__any(top > x.m)) {
        const float f = rescale(x.m, top);
        x.l *= f;
#pragma unroll
        for (int j = 0; j < kValues; ++j) x.acc[j] *= f;
        x.m = top;
      }
      const float base = (x.m == -INFINITY ? 0.0f : x.m) - (W::VT == kF16 ? 14.0f : 0.0f);
      float w[W::kSlots];
#pragma unroll
      for (int i = 0; i < W::kSlots; ++i) {
        w[i] = exp2_of(y[i] - base);
        x.l += w[i];
        if constexpr (CT == kE4M3) w[i] *= scale_v[i];
      }
      x.add_values(w);
      if (more) load_v(step + 1);
    }

    // the workgroup's waves: rows relative to the largest m
    const float l = query_sum(x.l);
    if (g == 0) {
      wave_ml[wave][0][c] = x.m;
      wave_ml[wave][1][c] = l;
    }
    const bool whole = u.first == 0 && u.last == u.tiles;
    const int64_t slot = 2 * (int64_t)blockIdx.x + (tile == share.begin ? 0 : 1);
    const int q = tid >> 4, r = tid & 15;  // a query, and the output rows r of the tiles
    const int64_t out_head = (int64_t)u.head * p.group + u.query_tile * 16 + q;
#pragma unroll
    for (int pass = 0; pass < kValues / kPass; ++pass) {
      if (pass > 0) __syncthreads();
      if (there) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < kPass; ++j) rows[wave][c * kRow + (4 * g + i) * kPass + j] = x.acc[pass * kPass + j][i];
      }
      __syncthreads();
      if (q < rows_here) {
        float top = -INFINITY, sum = 0.0f, f[kWaves];
#pragma unroll
        for (int i = 0; i < kWaves; ++i) top = fmaxf(top, wave_ml[i][0][q]);
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
          f[i] = rescale(wave_ml[i][0][q], top);
          sum += wave_ml[i][1][q] * f[i];
        }
        float o[kPass];
#pragma unroll
        for (int j = 0; j < kPass; ++j) {
          o[j] = 0.0f;
#pragma unroll
          for (int i = 0; i < kWaves; ++i) o[j] += rows[i][q * kRow + r * kPass + j] * f[i];
        }
        const int d0 = r * kValues + pass * kPass;
        constexpr float kShift = W::VT == kF16 ? 14.0f : 0.0f;
        if (whole) {
          T* out = reinterpret_cast<T*>(a.out) + u.seq * a.out_seq_stride + out_head * a.out_head_stride;
#pragma unroll
          for (int j = 0; j < kPass; ++j)
            if (EXACT || d0 + j < dim) out[d0 + j] = (T)(sum == 0.0f ? 0.0f : o[j] / sum);
          if (r == 0 && pass == 0) {
            const float all = sum == 0.0f ? -INFINITY : top - kShift + __builtin_amdgcn_logf(sum);
            if (a.lse) a.lse[u.seq * a.q_heads + out_head] = all * kLn2;
            if constexpr (ACC) p.sums[u.unit * 16 + q] = all;
          }
        } else {
          float* to = p.slot_rows + (slot * 16 + q) * DP + d0;
#pragma unroll
          for (int j = 0; j < kPass; ++j) to[j] = o[j];
          if (r == 0 && pass == 0) {
            p.slot_ml[slot * 32 + q] = top == -INFINITY ? top : top - kShift;
            p.slot_ml[slot * 32 + 16 + q] = sum;
          }
        }
      }
    }
    __syncthreads();  // the shared rows are free again

    tile = u.unit_tile + u.last;
    if (tile == seq_tile + u.tiles * p.units_per_seq) {
      seq_tile = tile;
      ++seq;
    }
  }
}

// ---------------------------------------------------------------------------
// the second kernel: joins the pieces of units, adds the attention weights
// ---------------------------------------------------------------------------
struct Pieces {
  int64_t first, last;  // workgroups that have tiles of the unit
  int64_t first_slot;   // of the first one; the others' is their first
  __device__ __forceinline__ int64_t slot(int64_t w) const { return w == first ? first_slot : 2 * w; }
};

__device__ __forceinline__ Pieces pieces_of(const Share& share, int64_t unit_tile, int64_t tiles) {
  Pieces r;
  r.first = share_of(share, unit_tile);
  r.last = share_of(share, unit_tile + tiles - 1);
  r.first_slot = 2 * r.first + (share_begin(share, r.first) == unit_tile ? 0 : 1);
  return r;
}

template <int QT, int DP, bool ACC>
__global__ __launch_bounds__(kThreads) void kv_join_kernel(const KvAttend a, const Plan p) {
  using T = kv_elem<QT>;
  __shared__ float part[kThreads];
  __shared__ float tops[16], all[16];
  const int tid = threadIdx.x;
  const KvPages& pages = a.pages;
  const int dim = pages.dim;
  const Share share = find_share(a, p);
  int64_t seq = share.seq, seq_tile = share.seq_tile;
  for (int64_t tile = share.begin; tile < share.end;) {
    const Piece u = piece_at(a, p, tile, share.end, seq, seq_tile);
    // m and log2 of the sum of all pieces of a unit of this sequence and head
    auto totals = [&](int query_tile, const Pieces& w) {
      const int q = tid >> 4, i0 = tid & 15;
      float top = -INFINITY;
      for (int64_t i = w.first + i0; i <= w.last; i += 16) top = fmaxf(top, p.slot_ml[w.slot(i) * 32 + q]);
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
      float sum = 0.0f;
      for (int64_t i = w.first + i0; i <= w.last; i += 16)
        sum += p.slot_ml[w.slot(i) * 32 + 16 + q] * rescale(p.slot_ml[w.slot(i) * 32 + q], top);
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
      __syncthreads();
      if (i0 == 0) {
        tops[q] = top;
        all[q] = sum == 0.0f ? -INFINITY : top + __builtin_amdgcn_logf(sum);
      }
      __syncthreads();
    };
    if (u.first != 0 || u.last != u.tiles) {
      const Pieces w = pieces_of(share, u.unit_tile, u.tiles);
      const int n = (int)(w.last - w.first + 1), me = (int)(blockIdx.x - w.first);
      const int rows_here = min(16, p.group - u.query_tile * 16);
      totals(u.query_tile, w);
      // this workgroup's run of the unit's output values
      const int e0 = (int)((int64_t)me * rows_here * dim / n), e1 = (int)((int64_t)(me + 1) * rows_here * dim / n);
      for (int e = e0; e < e1; e += kThreads) {
        const int width = min(e1 - e, kThreads), ways = kThreads / width;
        const int way = tid / width, mine = e + tid - way * width;
        float o = 0.0f;
        if (way < ways) {
          const int q = mine / dim, d = mine - q * dim;
          for (int64_t i = w.first + way; i <= w.last; i += ways)
            o += p.slot_rows[(w.slot(i) * 16 + q) * DP + d] * rescale(p.slot_ml[w.slot(i) * 32 + q], tops[q]);
        }
        __syncthreads();
        part[tid] = o;
        __syncthreads();
        if (way == 0) {
          for (int i = 1; i < ways; ++i) o += part[i * width + tid];
          const int q = mine / dim, d = mine - q * dim;
          const int64_t head = (int64_t)u.head * p.group + u.query_tile * 16 + q;
          const float sum = all[q] == -INFINITY ? 0.0f : exp2_of(tops[q] - all[q]);
          reinterpret_cast<T*>(a.out)[u.seq * a.out_seq_stride + head * a.out_head_stride + d] = (T)(o * sum);
        }
      }
      if (a.lse && me == 0 && tid < rows_here)
        a.lse[u.seq * a.q_heads + (int64_t)u.head * p.group + u.query_tile * 16 + tid] = all[tid] * kLn2;
      __syncthreads();
    }
    if constexpr (ACC) {
      // the first query tile's unit adds the weights of all query heads, so that no two add to one slot
      if (u.query_tile == 0) {
        const int64_t t0 = u.first * p.tile, t1 = min(u.last * p.tile, u.len);
        for (int qt = 0; qt < p.query_tiles; ++qt) {
          const int64_t unit_tile = u.unit_tile + qt * u.tiles;
          const Pieces w = pieces_of(share, unit_tile, u.tiles);
          if (w.first != w.last) {
            totals(qt, w);
          } else {
            __syncthreads();
            if (tid < 16) all[tid] = p.sums[(u.unit + qt) * 16 + tid];
            __syncthreads();
          }
          const int rows_here = min(16, p.group - qt * 16);
          const float* scores = p.scores + (u.seq * a.q_heads + (int64_t)u.head * p.group + qt * 16) * p.padded;
          for (int64_t t = t0 + tid; t < t1; t += kThreads) {
            const int64_t page = kv_page(pages, a.tables + u.seq * a.table_stride, t);
            if (page < 0) continue;
            float sum = 0.0f;
            for (int q = 0; q < rows_here; ++q)
              if (all[q] != -INFINITY) sum += exp2_of(scores[q * p.padded + t] - all[q]);
            pages.weights[kv_row(pages, page, u.head, t)] += sum;
          }
        }
        __syncthreads();
      }
    }
    tile = u.unit_tile + u.last;
    if (tile == seq_tile + u.tiles * p.units_per_seq) {
      seq_tile = tile;
      ++seq;
    }
  }
}

// A cache without pages: every sequence is empty.
template <int QT>
__global__ __launch_bounds__(kThreads) void kv_empty_kernel(const KvAttend a) {
  using T = kv_elem<QT>;
  const int64_t s = blockIdx.x;
  for (int i = threadIdx.x; i < a.q_heads * a.pages.dim; i += kThreads) {
    const int h = i / a.pages.dim, d = i - h * a.pages.dim;
    reinterpret_cast<T*>(a.out)[s * a.out_seq_stride + h * a.out_head_stride + d] = (T)0.0f;
    if (a.lse && d == 0) a.lse[s * a.q_heads + h] = -INFINITY;
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
int padded_dim(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

struct Layout {
  Plan plan;
  unsigned workgroups;
  size_t bytes;
};

Layout layout_of(const KvAttend& a, void* workspace) {
  Layout r{};
  Plan& p = r.plan;
  p.group = a.q_heads / a.pages.heads;
  p.query_tiles = (p.group + 15) / 16;
  p.units_per_seq = (int64_t)a.pages.heads * p.query_tiles;
  p.tile = tile_slots(a.dtype);
  const int64_t tiles = std::max<int64_t>(1, (a.max_length + p.tile - 1) / p.tile);
  const int64_t units = a.seqs * p.units_per_seq;
  p.padded = tiles * p.tile;
  const int dp = padded_dim(a.pages.dim);
  // resident workgroups: two on each of the 256 CUs
  const int64_t most = 512;
  r.workgroups = (unsigned)(units >= most ? most : std::min<int64_t>(most, units * tiles));
  uint8_t* at = static_cast<uint8_t*>(workspace);
  auto take = [&](size_t n) {
    float* x = reinterpret_cast<float*>(at + r.bytes);
    r.bytes += (n + 15) / 16 * 16;
    return x;
  };
  p.slot_rows = take((size_t)r.workgroups * 2 * 16 * dp * 4);
  p.slot_ml = take((size_t)r.workgroups * 2 * 32 * 4);
  if (a.accumulate) {
    p.sums = take((size_t)units * 16 * 4);
    p.scores = take((size_t)a.seqs * a.q_heads * p.padded * 4);
  }
  return r;
}

template <int QT, int CT, int DP, bool EXACT>
hipError_t launch_dim(const KvAttend& a, const Layout& l, hipStream_t stream) {
  if (a.pages.num_pages == 0) {
    kv_empty_kernel<QT><<<(unsigned)a.seqs, kThreads, 0, stream>>>(a);
    return hipGetLastError();
  }
  if (a.accumulate) {
    kv_attend_kernel<QT, CT, DP, EXACT, true><<<l.workgroups, kThreads, 0, stream>>>(a, l.plan);
    kv_join_kernel<QT, DP, true><<<l.workgroups, kThreads, 0, stream>>>(a, l.plan);
  } else {
    kv_attend_kernel<QT, CT, DP, EXACT, false><<<l.workgroups, kThreads, 0, stream>>>(a, l.plan);
    kv_join_kernel<QT, DP, false><<<l.workgroups, kThreads, 0, stream>>>(a, l.plan);
  }
  return hipGetLastError();
}

template <int QT, int CT>
hipError_t launch_types(const KvAttend& a, const Layout& l, hipStream_t stream) {
  const bool exact = a.pages.dim == padded_dim(a.pages.dim);
  switch (padded_dim(a.pages.dim)) {
    case 64: return exact ? launch_dim<QT, CT, 64, true>(a, l, stream) : launch_dim<QT, CT, 64, false>(a, l, stream);
    case 128:
      return exact ? launch_dim<QT, CT, 128, true>(a, l, stream) : launch_dim<QT, CT, 128, false>(a, l, stream);
    default:
      return exact ? launch_dim<QT, CT, 256, true>(a, l, stream) : launch_dim<QT, CT, 256, false>(a, l, stream);
  }
}

}  // namespace

size_t kv_attend_workspace(const KvAttend& a) { return a.seqs == 0 ? 0 : layout_of(a, nullptr).bytes; }

hipError_t launch_kv_attend(const KvAttend& a, void* workspace, hipStream_t stream) {
  if (a.seqs == 0) return hipSuccess;
  const Layout l = layout_of(a, workspace);
  const bool q8 = a.pages.dtype == kE4M3;
  switch (a.dtype) {
    case kF32: return launch_types<kF32, kF32>(a, l, stream);
    case kF16: return q8 ? launch_types<kF16, kE4M3>(a, l, stream) : launch_types<kF16, kF16>(a, l, stream);
    case kBF16: return q8 ? launch_types<kBF16, kE4M3>(a, l, stream) : launch_types<kBF16, kBF16>(a, l, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace nve_amd
