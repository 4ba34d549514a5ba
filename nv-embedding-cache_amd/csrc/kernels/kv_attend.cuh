// kv_attend.cuh -- attention of one new token per sequence over its pages: the kernels of all
// types, and their launches (instantiated by kv_attend.hip, and by kv_attend_mxfp4.hip for
// 4-bit pages).
//
// For a query head h and the slots t of its sequence: x_t = scale q . k_t,
// p = softmax(x), out = sum p_t v_t.  One pass over k and v with the running
// maximum m and sum l of the softmax; what was summed before is scaled by
// 2^(m_old - m) when the maximum grows (x in units of log2).
//
// Bound: every k and v row is read once, so the pages' bytes bound it; the matrix
// instructions keep the work per byte far below that for any group of up to 16 query
// heads that share a key head (larger groups read the rows once per 16).
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
// f32 has the same layout with 16 slots a step and products of one value a lane.
//
// Weights enter the second product as a sum of values of the product's type; one alone
// would lose as much as the output's own rounding, and the matrix units are idle
// anyway.  Three of bf16 hold all of an f32 weight, two of f16 22 bits of it.  All but
// the last are rounded towards zero and none is zero beside the first, so that all have
// the weight's sign and an infinite value gives an infinity, not a NaN.  e4m3 values,
// of 4 bits and never infinite, get two of bf16, each rounded to nearest: 17 bits
// (64 sequences of 2,000 slots of 64 values: 23.7 us, three 25.1).  f16 weights are
// held times 2^14, so that a long flat tail does not underflow (2^-38 of the
// maximum still counts).  e4m3 rows are widened exactly to the query's type
// (scores) and to bf16 (values); their scales go into scores and weights.
//
// Split.  A workgroup of 4 waves takes a run of tiles (4 kStep slots) of one unit, a
// (sequence, key head); its waves join through shared memory.  A unit that is one
// workgroup's is finished there; others leave f32 rows with their m and l in the
// workspace, and the second kernel joins them.  Weights are added by whoever knows
// a unit's sum: the first kernel for whole units, the second, piece by piece, for
// the others, from the scores that the first one left in the workspace.
//
//   Grid mode: a workgroup per piece of grid_chunk() tiles, as the tables' extent
//   asks for.  The unit is the fast index: consecutive workgroups go round the 8
//   XCDs, and later pieces exist for the long sequences only; with the piece as the
//   fast index (4 a unit) the first pieces met on two XCDs (64 sequences of 512 to
//   8,192 slots: 273 us, units first 183).
//   Stream mode, for tables far longer than their sequences: the machine's resident
//   workgroups share all tiles there are, units laid end to end, in equal runs.
// Two waves a SIMD at 128 values of 8 to 32 bits (one at 256, three at 64): k and v rows of the
// next step are in flight meanwhile, 32 KiB a workgroup.  Three were slower (one sequence
// of 200,001 slots: 170 us, two 146).
//
// 4-bit pages: a wave's step is 4.3 KB (128 values), a quarter of bf16's, so the work per slot counts, and more waves
// have to be under way: three a SIMD at 128 values.  Codes become bf16 with their scale in one instruction a pair
// (the conversion looks at nothing but a scale's exponent, so its byte is rotated into place and no more; the product
// that takes codes and scales as they are was 5e-5 of the largest sum off in 128 terms, too much).  The queries lie
// in shared memory, read in every step; the addresses of codes and exponents come from one row number.  One sequence of
// 400,001 slots, f16: 141 us with bf16's launch and two waves, 118 with output tiles two at a time, 106 with 512
// pieces, 97 with fewer registers, three waves and 768 pieces: 4.5 TB/s.  64 of 512 to 8,192 with weights: 87 to 79 us.
// Steps of 64 slots: 102 and 82 us.  f16 queries meet bf16 rows as two values of bf16, which hold all of their bits.
// The other widths (200,001 slots, bf16): 64 values 66 us with two, three or four waves, four taken, although with weights
// two take 51 us and three or four 70, as stream mode is slower with two (64 sequences of up to 2,000 slots: 28.5, four 25);
// four spill up to 12 registers in the kernels with weights, three of 32 values take 83 us for 64 of 512 to 8,192
// with weights, four 72.  256 values: two waves 93 us, one 110.
//
// Measured (bf16 / f16, 128 values, pages of 16): one sequence of 200,001 slots, 8 key
// heads: 144 us, 5.7 TB/s of the pages' bytes (a large copy moves 4.7 TB/s, read and
// written); 64 sequences of 512 to 8,192 slots with weights: 181 us (165 and 15 in the
// two kernels), 4.1 TB/s; 256 of 200 to 4,096 in e4m3, 8 queries a key head: 157 us, 4.5 TB/s.
// One of 777 slots: 9.8 us, two launches of three dependent reads each.
#pragma once

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

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// f32 has 4 slots per lane and step, the other types 8.
constexpr int step_slots(int qt) { return qt == kF32 ? 16 : 32; }

// ---------------------------------------------------------------------------
// the workgroups' tiles
// ---------------------------------------------------------------------------
// A unit is a (sequence, key head); a piece a run of its tiles in one workgroup.
struct Plan {
  int32_t query_tiles, group, tile;
  int32_t chunk, pieces;  // grid mode: tiles of a piece (0: by the length), pieces of a unit at most
  int32_t workgroups;     // stream mode
  // Scores in log2 units (accumulate): rows of score_row floats, one per query head of the call
  // with its sequence's slots in order, or (by_slot) one per query of a group with the cache's
  // slots as the weights have them.
  int32_t by_slot;
  int64_t score_row;
  float* scores;
  float* slot_ml;         // [slots, query_tiles, 2, 16]
  float* slot_rows;       // [slots, query_tiles, 16, dim padded]
  struct Slot* slots;     // [2 * workgroups] (stream mode)
};

struct Piece {
  int seq, head, tiles;  // the unit and its number of tiles
  int first, last;       // [first, last) of them
  int64_t len;           // the sequence's
};

// What a stream workgroup leaves of the first and the last piece of its share.
struct Slot {
  int32_t valid, unit_tile, total;
  Piece piece;
};

// The same in every lane, and so in a scalar register: what describes a share must not
// take vector registers from the loop over its tiles.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Tiles of a sequence; one at least, so that an empty one is visited.
__device__ __forceinline__ int tiles_of(const Plan& p, int64_t len) {
  return len <= p.tile ? 1 : (int)((len + p.tile - 1) / p.tile);
}

// Grid mode: tiles of a unit's pieces.
__device__ __forceinline__ int chunk_of(const Plan& p, int tiles) {
  return p.chunk > 0 ? p.chunk : (tiles + p.pieces - 1) / p.pieces;
}

// Stream mode: all tiles of the call, end to end, in shares that differ by one tile at most.
struct Shares {
  int total, workers;  // no share is empty
  int base, more;      // the first `more` shares have base + 1 tiles
  __device__ __forceinline__ Shares(int total, int workgroups) : total(total) {
    workers = total < workgroups ? total : workgroups;
    base = total / workers;
    more = total - base * workers;
  }
  __device__ __forceinline__ int begin(int w) const { return w * base + (w < more ? w : more); }
  __device__ __forceinline__ int of(int tile) const {  // the share a tile is in
    const int long_end = more * (base + 1);
    return tile < long_end ? tile / (base + 1) : more + (tile - long_end) / base;
  }
};

struct Start {
  int total;
  int seq, seq_tile;  // the sequence that the share starts in, and the call's tile where that starts
};

// Every thread sums a run of the sequences; a scan finds where this workgroup's share starts.
__device__ __forceinline__ Start find_start(const KvAttend& a, const Plan& p) {
  __shared__ int wave_total[4];
  __shared__ int found[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int seqs = (int)a.seqs, per = (seqs + 255) / 256;
  const int s0 = min(per * tid, seqs), s1 = min(s0 + per, seqs);
  int own = 0;
  for (int s = s0; s < s1; ++s) own += tiles_of(p, kv_length(a.lengths, s, a.max_length));
  int scan = own;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(scan, d);
    if (lane >= d) scan += o;
  }
  if (lane == 63) wave_total[wave] = scan;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wave) scan += wave_total[w];
    total += wave_total[w];
  }
  Start r;
  r.total = uniform(total * a.pages.heads);
  const Shares shares(r.total, p.workgroups);
  const int begin = (int)blockIdx.x < shares.workers ? shares.begin(blockIdx.x) : r.total;
  int at = (scan - own) * a.pages.heads;
  if (begin >= at && begin < scan * a.pages.heads) {
    int s = s0;
    for (; s + 1 < s1; ++s) {
      const int n = tiles_of(p, kv_length(a.lengths, s, a.max_length)) * a.pages.heads;
      if (begin < at + n) break;
      at += n;
    }
    found[0] = s;
    found[1] = at;
  }
  __syncthreads();
  r.seq = uniform(found[0]);
  r.seq_tile = uniform(found[1]);
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
// Rounded towards zero.
template <int QT>
__device__ __forceinline__ uint32_t pack2_down(float a, float b) {
  if constexpr (QT == kF16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
  else
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
// The type's least positive value in place of a zero beside a high half that is none.
__device__ __forceinline__ uint32_t at_least_one(uint32_t low, uint32_t high) {
  using u16x2 = __attribute__((ext_vector_type(2))) uint16_t;
  const u16x2 one = {1, 1};
  return __builtin_bit_cast(uint32_t,
                            __builtin_elementwise_max(__builtin_bit_cast(u16x2, low),
                                                      __builtin_elementwise_min(__builtin_bit_cast(u16x2, high), one)));
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
template <int QT>
__device__ __forceinline__ uint32_t widen2(uint32_t w, bool high) {
  if constexpr (QT == kF16)
    return __builtin_bit_cast(uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true)
                                             : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
  else
    return __builtin_bit_cast(uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true)
                                             : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
}

// Two of 8 e2m1 codes, the first one lowest, times their scale: exact in bf16.
__device__ __forceinline__ uint32_t widen_pair(uint32_t w, float scale, int pair) {
  switch (pair) {
    case 0: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
    case 1: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
    case 2: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
    default: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
  }
}
__device__ __forceinline__ u32x4 widen8(uint32_t w, float scale) {
  return u32x4{widen_pair(w, scale, 0), widen_pair(w, scale, 1), widen_pair(w, scale, 2), widen_pair(w, scale, 3)};
}
// The scale of an exponent byte; 255 is a NaN's place, and the conversions give NaN for it.
__device__ __forceinline__ float block_scale(uint32_t e) { return __uint_as_float(e << 23); }
__device__ __forceinline__ uint32_t load_byte(const uint8_t* p) {
  return *(const __attribute__((address_space(1))) uint8_t*)(uintptr_t)p;
}

// 4 to 16 bytes of a row (any 4-byte alignment).
template <int N>
using words = __attribute__((ext_vector_type(N))) uint32_t;

template <int N>
__device__ __forceinline__ words<N> load_words(const uint8_t* src) {
  typedef words<N> __attribute__((aligned(4))) any;
  return *(const __attribute__((address_space(1))) any*)(uintptr_t)src;
}

// The first row of scores of a unit's query tile.
__device__ __forceinline__ int64_t score_row_of(const KvAttend& a, const Plan& p, const Piece& u, int query_tile) {
  return (p.by_slot ? 0 : u.seq * (int64_t)a.q_heads + (int64_t)u.head * p.group) + query_tile * 16;
}

// The weights of a piece's slots under `rows` softmaxes whose sums are all[]; four slots a
// thread, which lie in one page.
__device__ __forceinline__ void add_weights(const KvAttend& a, const Plan& p, const Piece& u, int query_tile,
                                            const float* all) {
  typedef f32x4 __attribute__((aligned(4))) f4;
  const int64_t t1 = min((int64_t)u.last * p.tile, u.len);
  const int rows = min(16, p.group - query_tile * 16);
  const float* scores = p.scores + score_row_of(a, p, u, query_tile) * p.score_row;
  for (int64_t t = (int64_t)u.first * p.tile + 4 * threadIdx.x; t < t1; t += 4 * 256) {
    const int64_t page = kv_page(a.pages, a.tables + u.seq * a.table_stride, t);
    if (page < 0) continue;
    const int64_t row = kv_row(a.pages, page, u.head, t), at = p.by_slot ? row : t;
    float* to = a.pages.weights + row;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int q0 = 0; q0 < rows; q0 += 4) {  // four rows' loads together
      f32x4 x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = *reinterpret_cast<const f32x4*>(scores + min(q0 + j, rows - 1) * p.score_row + at);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // an empty softmax has no weights, nor has a row past the last
        const float y = q0 + j >= rows || all[q0 + j] == -INFINITY ? INFINITY : all[q0 + j];
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] += exp2_of(x[j][i] - y);
      }
    }
    if (t + 4 <= t1) {
      *reinterpret_cast<f4*>(to) += sum;
    } else {
      for (int i = 0; i < (int)(t1 - t); ++i) to[i] += sum[i];
    }
  }
}

// ---------------------------------------------------------------------------
// the first kernel
// ---------------------------------------------------------------------------
// DP: head_dim rounded up to 64, 128 or 256; EXACT: head_dim is DP.
template <int QT, int CT, int DP, bool EXACT>
struct Wave {
  static constexpr bool k4 = CT == kMXFP4;
  static constexpr bool kCoded = CT == kE4M3 || k4;  // few bits a value and never infinite
  static constexpr int kStep = step_slots(QT);
  static constexpr int kTiles = kStep / 16;        // score tiles of a step
  static constexpr int kSlots = kStep / 4;         // slots of a lane
  static constexpr int kRowBytes = kv_row_bytes(CT, DP);
  static constexpr int kPieces = kRowBytes < 64 ? 1 : kRowBytes / 64;  // 16-byte pieces of a k row in a lane
  static constexpr int kRun = 32 / (256 / DP > 2 ? 2 : 1);  // 4 bits: neighbours of a k row in a lane
  static constexpr int kSteps = DP / 32;           // 16-bit products of a row
  static constexpr int kValues = DP / 16;          // values of a v row in a lane, and output tiles
  static constexpr int kVWords = (kRowBytes / 16 + 3) / 4;
  static constexpr int VT = kCoded ? kBF16 : QT;  // the type of the second product
  static constexpr int kParts = CT == kBF16 ? 3 : 2;    // of a weight
  static constexpr int kQWords = QT == kF32 ? DP / 4 : kSteps * 4;
  static constexpr int kQParts = k4 && QT == kF16 ? 2 : 1;  // queries meet 4-bit rows in bf16

  static constexpr int kVLoad = !EXACT && CT == kE4M3 ? (kVWords < 2 ? 1 : 2) : kVWords < 4 ? kVWords : 4;

  u32x4 q[k4 ? 1 : kQParts][k4 ? 1 : kQWords / 4];  // 4 bits: in shared memory
  u32x4 k[kTiles][kPieces];
  words<kVLoad> v[kSlots][kVWords / kVLoad];
  f32x4 k_scale[kTiles], v_scale[kTiles];  // e4m3: of this lane's slots
  // 4 bits: exponents, of this lane's k pieces, and of its slots' v rows: those of the lane's values, or
  // (kRowWords dwords for four rows) of all
  static constexpr int kRowWords = k4 && EXACT && DP <= 128 ? DP / 32 : 0;
  uint32_t k_block[kTiles][kPieces], v_block[kSlots];
  uint32_t v_words[kTiles][kRowWords > 0 ? kRowWords : 1];
  f32x4 acc[kValues];
  float m, l;  // m: of the query; l: of this lane's slots

  // The value of a row where word w of a lane's queries starts.
  static __device__ __forceinline__ int q_value(int w, int g) {
    if constexpr (QT == kF32) return (w >> 2) * 16 + g * 4 + (w & 3);
    const int step = w >> 2, i = (w & 3) * 2;
    if constexpr (k4) return step * 8 / kRun * (4 * kRun) + g * kRun + step * 8 % kRun + i;
    if constexpr (CT == kE4M3) return (step >> 1) * 64 + g * 16 + (step & 1) * 8 + i;
    return step * 32 + g * 8 + i;
  }

  // Queries may start at any element: 16-byte loads of the type's alignment.
  __device__ __forceinline__ void load_queries(const KvAttend& a, int64_t row_offset, bool there, int g,
                                               u32x4 (*shared)[64]) {
    constexpr int kElem = QT == kF32 ? 4 : 2;
    typedef u32x4 __attribute__((aligned(2))) any4;
    const int dim = a.pages.dim;
    // 4 bits: all waves have the same queries, and each brings a part of them
#pragma unroll
    for (int w = 0; w < kQWords; w += 4) {
      if (k4 && (w / 4) % 4 != (int)(threadIdx.x >> 6)) continue;
      const int d = q_value(w, g);
      u32x4 x = {0, 0, 0, 0};
      if (there && (EXACT || d < dim)) x = *reinterpret_cast<const any4*>(a.q.p + (row_offset + d) * kElem);
      if constexpr (k4) {
        u32x4 rest = {0, 0, 0, 0};
        if constexpr (kQParts == 2) {  // 11 bits are 8 and 3
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float u = low_of<kF16>(x[i]), v = high_of<kF16>(x[i]);
            const uint32_t h = pack2<kBF16>(u, v);
            x[i] = h;
            rest[i] = pack2<kBF16>(u - low_of<kBF16>(h), v - high_of<kBF16>(h));
          }
          shared[kQWords / 4 + w / 4][threadIdx.x & 63] = rest;
        }
        shared[w / 4][threadIdx.x & 63] = x;
      } else {
        q[0][w / 4] = x;
      }
    }
  }

  // A k row's pieces: 16 bytes at 64 i + 16 g.
  static __device__ __forceinline__ void load_k(u32x4 (&r)[kPieces], const uint8_t* row, int g, int dim) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int b = i * 64 + g * 16;
      if constexpr (k4 && DP == 64) {
        words<2> x = {0, 0};
        if (EXACT || g * kRun < dim) x = load_words<2>(row + g * 8);
        r[i] = u32x4{x[0], x[1], 0, 0};
      } else if constexpr (k4) {
        r[i] = u32x4{0, 0, 0, 0};
        if (EXACT || b < dim / 2) r[i] = load_words<4>(row + b);
      } else if constexpr (EXACT) {
        r[i] = load_words<4>(row + b);
      } else if constexpr (CT == kE4M3) {  // head_dim is a multiple of 8: half a piece
        words<2> low = {0, 0}, high = {0, 0};
        if (b < dim) low = load_words<2>(row + b);
        if (b + 8 < dim) high = load_words<2>(row + b + 8);
        r[i] = u32x4{low[0], low[1], high[0], high[1]};
      } else {
        r[i] = u32x4{0, 0, 0, 0};
        if (b < kv_row_bytes(CT, dim)) r[i] = load_words<4>(row + b);
      }
    }
  }

  // 4 bits: the exponents of a k row's pieces, and of a v row's values.
  static __device__ __forceinline__ void load_k_blocks(uint32_t (&e)[kPieces], const uint8_t* blocks, int g, int dim) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int d = i * 4 * kRun + g * kRun;
      e[i] = 127;
      if (EXACT || d < dim) e[i] = load_byte(blocks + d / 32);
    }
  }
  static __device__ __forceinline__ void load_v_words(uint32_t (&w)[kRowWords > 0 ? kRowWords : 1], const uint8_t* blocks) {
    typedef u32x4 __attribute__((aligned(1))) any4;
    typedef words<2> __attribute__((aligned(1))) any2;
    if constexpr (kRowWords == 4) {
      const u32x4 x = *(const __attribute__((address_space(1))) any4*)(uintptr_t)blocks;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = x[i];
    } else {
      const words<2> x = *(const __attribute__((address_space(1))) any2*)(uintptr_t)blocks;
      w[0] = x[0];
      w[1] = x[1];
    }
  }
  // The scale of a slot's values.  The conversions look at a scale's exponent alone, so the byte is rotated there
  // and what is beside it stays.
  __device__ __forceinline__ float v_scale_of(int slot, int c) const {
    if constexpr (kRowWords == 0) return block_scale(v_block[slot]);
    const uint32_t w = v_words[slot / 4][slot % 4 * kRowWords / 4];
    const uint32_t byte = slot % 4 * kRowWords % 4 + c * kValues / 32;
    return __uint_as_float(__builtin_amdgcn_alignbit(w, w, 8 * byte + 9));
  }
  static __device__ __forceinline__ uint32_t load_v_block(const uint8_t* blocks, int c, int dim) {
    const int d = c * kValues;
    return load_byte(blocks + (EXACT || d < dim ? d / 32 : 0));
  }

  // A v row's values kValues c ..; those past head_dim are not used (the row's first instead).
  static __device__ __forceinline__ void load_v(words<kVLoad> (&r)[kVWords / kVLoad], const uint8_t* row, int c, int dim) {
    const int b = c * kRowBytes / 16;
    if constexpr (k4 && DP == 64) {
      r[0][0] = *(const __attribute__((address_space(1))) uint16_t*)(uintptr_t)(row + (EXACT || b < dim / 2 ? b : 0));
      return;
    }
#pragma unroll
    for (int i = 0; i < kVWords / kVLoad; ++i) {
      const int at = b + 4 * kVLoad * i;
      r[i] = load_words<kVLoad>(row + (EXACT || at < kv_row_bytes(CT, dim) ? at : 0));
    }
  }

  // 4 bits: of all tiles of a step, each read of the queries for all.
  __device__ __forceinline__ void scores4(f32x4 (&s)[kTiles], const u32x4 (*shared)[64]) const {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));  // read again in every step, and not kept in registers through the loop
#pragma unroll
    for (int n = 0; n < kTiles; ++n) s[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      u32x4 y[kQParts];
#pragma unroll
      for (int h = 0; h < kQParts; ++h) y[h] = shared[h * kSteps + i][lane];
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        const int piece = i * 8 / kRun;
        const u32x4 x = widen8(k[n][piece][i * 8 % kRun / 8], block_scale(k_block[n][piece]));
#pragma unroll
        for (int h = 0; h < kQParts; ++h) s[n] = mma<kBF16>(x, y[h], s[n]);
      }
    }
  }

  __device__ __forceinline__ f32x4 scores(int tile) const {
    f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (QT == kF32) {
#pragma unroll
      for (int w = 0; w < DP / 4; ++w)
        s = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[tile][w / 4][w % 4]), __uint_as_float(q[0][w / 4][w % 4]), s,
                                                  0, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        u32x4 x;
        if constexpr (CT == kE4M3) {
          const uint32_t w0 = k[tile][i / 2][i % 2 * 2], w1 = k[tile][i / 2][i % 2 * 2 + 1];
          x = u32x4{widen2<QT>(w0, false), widen2<QT>(w0, true), widen2<QT>(w1, false), widen2<QT>(w1, true)};
        } else {
          x = k[tile][i];
        }
        s = mma<QT>(x, q[0][i], s);
      }
    }
    return s;
  }

  // acc += V^T P^T for the weights p of this lane's slots.
  __device__ __forceinline__ void add_values(const float (&p)[kSlots], int c) {
    if constexpr (QT == kF32) {
#pragma unroll
      for (int j = 0; j < kValues; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[r][j / kVLoad][j % kVLoad]), p[r], acc[j], 0, 0, 0);
    } else {
      u32x4 part[kParts];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float a = p[2 * i], b = p[2 * i + 1];
#pragma unroll
        for (int n = 0; n < kParts; ++n) {
          const bool last = n == kParts - 1;
          const uint32_t w = kCoded || (last && VT == kF16) ? pack2<VT>(a, b) : pack2_down<VT>(a, b);
          a -= low_of<VT>(w);
          b -= high_of<VT>(w);
          part[n][i] = kCoded || n == 0 ? w : at_least_one(w, part[0][i]);
        }
      }
      if constexpr (k4) {
        // two output tiles at a time, so that few widened values are alive
        float scale[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) scale[r] = v_scale_of(r, c);
#pragma unroll
        for (int j = 0; j < kValues; j += 2) {
          uint32_t w[8];
#pragma unroll
          for (int r = 0; r < 8; ++r) w[r] = widen_pair(v[r][j / 8 / kVLoad][j / 8 % kVLoad], scale[r], j / 2 % 4);
          u32x4 x, y;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x05040100u);
            y[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x07060302u);
          }
#pragma unroll
          for (int n = 0; n < kParts; ++n) {
            acc[j] = mma<VT>(x, part[n], acc[j]);
            acc[j + 1] = mma<VT>(y, part[n], acc[j + 1]);
          }
        }
        return;
      }
      uint32_t w[8][kValues / 2];
#pragma unroll
      for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int i = 0; i < kValues / 2; ++i) {
          if constexpr (CT == kE4M3)
            w[r][i] = widen2<VT>(v[r][i / 2 / kVLoad][i / 2 % kVLoad], i & 1);
          else
            w[r][i] = v[r][i / kVLoad][i % kVLoad];
        }
#pragma unroll
      for (int j = 0; j < kValues; ++j) {
        u32x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[i] = __builtin_amdgcn_perm(w[2 * i + 1][j / 2], w[2 * i][j / 2], (j & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int n = 0; n < kParts; ++n) acc[j] = mma<VT>(x, part[n], acc[j]);
      }
    }
  }
};

// Waves of a SIMD (and workgroups of a CU) that the kernel is built for and stream mode fills.
constexpr int waves_per_simd(int ct, int dp) {
  if (ct == kMXFP4) return dp == 64 ? 4 : dp == 128 ? 3 : 2;
  return dp == 64 ? 3 : dp == 128 ? 2 : 1;
}

template <int QT, int CT, int DP, bool EXACT, bool ACC, bool GRID>
__global__ __launch_bounds__(256, waves_per_simd(CT, DP)) void kv_attend_kernel(const KvAttend a, const Plan p) {
  using W = Wave<QT, CT, DP, EXACT>;
  using T = kv_elem<QT>;
  constexpr int kWaves = 4, kStep = W::kStep, kValues = W::kValues;
  constexpr int kPass = 4;            // output tiles joined at a time
  constexpr int kRow = 16 * kPass + 4;  // a query's values in shared memory, padded
  __shared__ float wave_ml[kWaves][2][16];
  __shared__ float rows[kWaves][16 * kRow];
  __shared__ float all[16];
  __shared__ u32x4 queries[W::k4 ? W::kQParts * W::kSteps : 1][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = W::k4 ? uniform(tid >> 6) : tid >> 6, c = lane & 15, g = lane >> 4;
  const KvPages& pages = a.pages;
  const int dim = EXACT ? DP : pages.dim;
  const int row_bytes = kv_row_bytes(CT, dim), mask = pages.page - 1;
  const uint64_t page_bytes = (uint64_t)pages.heads * pages.page * row_bytes;
  const float to_log2 = a.scale * kLog2e;
  W x;

  // One piece and 16 of its queries; the slot is where it goes if the unit has others.
  auto process = [&](const Piece& u, int query_tile, int slot) {
    const int rows_here = min(16, p.group - query_tile * 16);
    const int64_t q_head = (int64_t)u.head * p.group + query_tile * 16 + c;
    const bool there = c < rows_here;
    x.load_queries(a, u.seq * a.q.token_stride + q_head * a.q.head_stride, there, g, queries);
    if constexpr (W::k4) __syncthreads();
#pragma unroll
    for (int j = 0; j < kValues; ++j) x.acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    x.m = -INFINITY;
    x.l = 0.0f;

    float* score_row = nullptr;  // of this lane's query
    if constexpr (ACC) score_row = p.scores + (score_row_of(a, p, u, query_tile) + c) * p.score_row;
    const int32_t* table = a.tables + u.seq * a.table_stride;
    const int steps = u.last - u.first;
    const int64_t t_base = (int64_t)u.first * (kWaves * kStep) + wave * kStep;  // this wave's first slot
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
    auto scale_at = [&](const void* base, int id, int64_t t) {
      typedef f32x4 __attribute__((aligned(4))) f4;
      return *reinterpret_cast<const f4*>(static_cast<const float*>(base) +
                                          ((int64_t)max(id, 0) * pages.heads + u.head) * pages.page + (t & mask));
    };
    // 4 bits: a row's number in the cache, for its codes and its exponents, from what all lanes have (the tile's first
    // slot) and what is a lane's own.
    auto row_number = [&](int id, int64_t tile_t, int in_tile) {
      const uint32_t in_page = (uint32_t)(u.head * pages.page + ((int)tile_t & mask)) + (uint32_t)(in_tile & mask);
      return (uint64_t)(uint32_t)max(id, 0) * (uint32_t)(pages.heads * pages.page) + in_page;
    };
    // Slots without a row read the first page's instead; their scores and values are dropped below.
    auto load_k = [&](int step) {
      const int64_t t0 = t_base + (int64_t)step * (kWaves * kStep);
#pragma unroll
      for (int n = 0; n < W::kTiles; ++n) {
        const int id = __shfl(ids, (step & 15) * 4 + n * 2 + (c >> 3));
        if constexpr (W::k4) {
          const uint64_t row = row_number(id, t0 + n * 16, c);
          W::load_k(x.k[n], pages.k + row * row_bytes, g, dim);
          W::load_k_blocks(x.k_block[n], static_cast<const uint8_t*>(pages.k_scale) + row * (dim / 32), g, dim);
        } else {
          W::load_k(x.k[n], row_at(pages.k, id, t0 + n * 16 + c), g, dim);
        }
        if constexpr (CT == kE4M3) {
          const int of = __shfl(ids, (step & 15) * 4 + n * 2 + (g >> 1));
          x.k_scale[n] = scale_at(pages.k_scale, of, t0 + n * 16 + g * 4);
        }
      }
    };
    auto load_v = [&](int step) {
      const int64_t t0 = t_base + (int64_t)step * (kWaves * kStep);
#pragma unroll
      for (int n = 0; n < W::kTiles; ++n) {
        const int id = __shfl(ids, (step & 15) * 4 + n * 2 + (g >> 1));
        const int64_t t = t0 + n * 16 + g * 4;
        const uint64_t number = W::k4 ? row_number(id, t0 + n * 16, g * 4) : 0;
        const uint8_t* row = W::k4 ? pages.v + number * row_bytes : row_at(pages.v, id, t);
#pragma unroll
        for (int r = 0; r < 4; ++r) W::load_v(x.v[n * 4 + r], row + r * row_bytes, c, dim);
        if constexpr (CT == kE4M3) x.v_scale[n] = scale_at(pages.v_scale, id, t);
        if constexpr (W::k4) {
          const uint8_t* blocks = static_cast<const uint8_t*>(pages.v_scale) + number * (dim / 32);
          if constexpr (W::kRowWords > 0) {
            W::load_v_words(x.v_words[n], blocks);
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) x.v_block[n * 4 + r] = W::load_v_block(blocks + r * (dim / 32), c, dim);
          }
        }
      }
    };

    load_ids(0);
    load_k(0);
    load_v(0);
    // A step; with `more` the next one's rows are requested on the way.  The last step is apart,
    // because a wait after a branch around loads has to suit the path without them: it would wait
    // for the next step's rows as well.
    auto advance = [&](int step, auto more) {
      const int64_t t0 = t_base + (int64_t)step * (kWaves * kStep);
      f32x4 s[W::kTiles];
      if constexpr (W::k4) {
        x.scores4(s, queries);
      } else {
#pragma unroll
        for (int n = 0; n < W::kTiles; ++n) s[n] = x.scores(n);
      }
      // the four page numbers of this step, -1 where a slot has no row
      const uint64_t absent = __ballot(ids < 0) >> ((step & 15) * 4);
      const bool full = t0 + kStep <= u.len && (absent & (kStep == 32 ? 15 : 3)) == 0;
      float y[W::kSlots];
#pragma unroll
      for (int n = 0; n < W::kTiles; ++n) {
        const int id = __shfl(ids, (step & 15) * 4 + n * 2 + (g >> 1));
        const int64_t t = t0 + n * 16 + g * 4;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          y[n * 4 + r] = s[n][r] * to_log2;
          if constexpr (CT == kE4M3) y[n * 4 + r] *= x.k_scale[n][r];
        }
        if (!full) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool row = id >= 0 && t + r < u.len;
            const uint32_t keep = row ? 0xffffffffu : 0u;
            y[n * 4 + r] = row ? y[n * 4 + r] : -INFINITY;
            if constexpr (CT == kE4M3) x.v_scale[n][r] = row ? x.v_scale[n][r] : 0.0f;
            if constexpr (W::kRowWords > 0) {  // no NaN beside the codes, which become 0
              const uint32_t bytes = W::kRowWords == 4 ? 0xffffffffu : 0xffffu << (16 * (r & 1));
              x.v_words[n][r * W::kRowWords / 4] &= keep | ~bytes;
            } else if constexpr (W::k4) {
              x.v_block[n * 4 + r] &= keep;
            }
#pragma unroll
            for (int w = 0; w < W::kVWords / W::kVLoad; ++w) x.v[n * 4 + r][w] &= keep;
          }
        }
        if constexpr (ACC) {
          if (there && id >= 0 && t < u.len) {  // rows of scores are padded to whole tiles or pages
            const int64_t at = p.by_slot ? kv_row(pages, id, u.head, t) : t;
            *reinterpret_cast<f32x4*>(score_row + at) = f32x4{y[n * 4], y[n * 4 + 1], y[n * 4 + 2], y[n * 4 + 3]};
          }
        }
      }
      if constexpr (more) {
        if (((step + 1) & 15) == 0) load_ids(step + 1);
        load_k(step + 1);
      }

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
        if constexpr (CT == kE4M3) w[i] *= x.v_scale[i / 4][i % 4];
      }
      x.add_values(w, c);
      if constexpr (more) load_v(step + 1);
    };
    for (int step = 0; step + 1 < steps; ++step) advance(step, std::true_type());
    advance(steps - 1, std::false_type());

    // the workgroup's waves: rows relative to the largest m.  4 bits: what only this needs is worked out here, and
    // not held in registers through the loop above.
    int end_tid = tid;
    if constexpr (W::k4) asm volatile("" : "+v"(end_tid));
    const int end_wave = W::k4 ? end_tid >> 6 : wave, end_c = W::k4 ? end_tid & 15 : c, end_g = W::k4 ? (end_tid >> 4) & 3 : g;
    const float l = query_sum(x.l);
    if (end_g == 0) {
      wave_ml[end_wave][0][end_c] = x.m;
      wave_ml[end_wave][1][end_c] = l;
    }
    const bool whole = u.first == 0 && u.last == u.tiles;
    const int q = end_tid >> 4, r = end_tid & 15;  // a query, and the output rows r of the tiles
    const int64_t out_head = (int64_t)u.head * p.group + query_tile * 16 + q;
    const int64_t at = (int64_t)slot * p.query_tiles + query_tile;
#pragma unroll
    for (int pass = 0; pass < kValues / kPass; ++pass) {
      if (pass > 0) __syncthreads();
      if (there) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < kPass; ++j) rows[end_wave][end_c * kRow + (4 * end_g + i) * kPass + j] = x.acc[pass * kPass + j][i];
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
            const float log_sum = sum == 0.0f ? -INFINITY : top - kShift + __builtin_amdgcn_logf(sum);
            if (a.lse) a.lse[u.seq * a.q_heads + out_head] = log_sum * kLn2;
            all[q] = log_sum;
          }
        } else {
          float* to = p.slot_rows + (at * 16 + q) * DP + d0;
#pragma unroll
          for (int j = 0; j < kPass; ++j) to[j] = o[j];
          if (r == 0 && pass == 0) {
            p.slot_ml[at * 32 + q] = top == -INFINITY ? top : top - kShift;
            p.slot_ml[at * 32 + 16 + q] = sum;
          }
        }
      }
    }
    if (ACC && whole) {
      __threadfence_block();  // the other waves' scores
      __syncthreads();
      add_weights(a, p, u, query_tile, all);
    }
    __syncthreads();  // the shared rows are free again
  };

  if constexpr (GRID) {
    const int unit = blockIdx.x;  // units first: their pieces, of which there may be fewer, spread over the XCDs
    Piece u;
    u.seq = unit / pages.heads;
    u.head = unit - u.seq * pages.heads;
    u.len = kv_length(a.lengths, u.seq, a.max_length);
    u.tiles = tiles_of(p, u.len);
    const int chunk = chunk_of(p, u.tiles);
    u.first = blockIdx.y * chunk;
    u.last = min(u.first + chunk, u.tiles);
    if (u.first >= u.tiles) return;
    for (int qt = 0; qt < p.query_tiles; ++qt) process(u, qt, unit * p.pieces + blockIdx.y);
  } else {
    const Start start = find_start(a, p);
    const Shares shares(start.total, p.workgroups);
    const int w = blockIdx.x;
    if (tid == 0) p.slots[2 * w].valid = p.slots[2 * w + 1].valid = 0;
    if (w >= shares.workers) return;
    const int begin = shares.begin(w), end = shares.begin(w + 1);
    int seq = start.seq, seq_tile = start.seq_tile;
    for (int tile = begin; tile < end;) {
      Piece u;
      u.seq = seq;
      u.len = kv_length(a.lengths, seq, a.max_length);
      u.tiles = tiles_of(p, u.len);
      u.head = (tile - seq_tile) / u.tiles;
      const int unit_tile = seq_tile + u.head * u.tiles;
      u.first = tile - unit_tile;
      u.last = min(end - unit_tile, u.tiles);
      const int slot = 2 * w + (tile == begin ? 0 : 1);
      if (tid == 0 && !(u.first == 0 && u.last == u.tiles)) p.slots[slot] = Slot{1, unit_tile, start.total, u};
      for (int qt = 0; qt < p.query_tiles; ++qt) process(u, qt, slot);
      tile = unit_tile + u.last;
      if (tile == seq_tile + u.tiles * pages.heads) {
        seq_tile = tile;
        ++seq;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// the second kernel: joins the pieces of units, adds the attention weights
// ---------------------------------------------------------------------------
// A unit's pieces: in grid mode slots in a row, in stream mode the slots of the workgroups
// that have its tiles (the first one's `head`, then each one's first).
struct Pieces {
  int count, head, next, step;
  __device__ __forceinline__ int slot(int i) const { return i == 0 ? head : next + (i - 1) * step; }
};

// The largest m of a unit's pieces, and log2 of the sum over all of them, for 16 queries.
__device__ __forceinline__ void total_of(const Plan& p, const Pieces& w, int query_tile, float* tops, float* all) {
  constexpr int kAhead = 8;
  const int q = threadIdx.x >> 4, lane = threadIdx.x & 15;
  float top = -INFINITY, sum = 0.0f;
  for (int i0 = lane; i0 < w.count; i0 += 16 * kAhead) {
    float m[kAhead], l[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int i = i0 + 16 * j;
      m[j] = -INFINITY;
      l[j] = 0.0f;
      if (i < w.count) {
        const float* ml = p.slot_ml + ((int64_t)w.slot(i) * p.query_tiles + query_tile) * 32 + q;
        m[j] = ml[0];
        l[j] = ml[16];
      }
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const float t = fmaxf(top, m[j]);
      sum = sum * rescale(top, t) + l[j] * rescale(m[j], t);
      top = t;
    }
  }
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) {
    const float m = __shfl_xor(top, d), l = __shfl_xor(sum, d);
    const float t = fmaxf(top, m);
    sum = sum * rescale(top, t) + l * rescale(m, t);
    top = t;
  }
  __syncthreads();
  if (lane == 0) {
    tops[q] = top;
    all[q] = sum == 0.0f ? -INFINITY : top + __builtin_amdgcn_logf(sum);
  }
  __syncthreads();
}

constexpr int kJoinValues = 64;  // output values a joining workgroup has at least

template <int QT, int DP, bool ACC, bool GRID>
__global__ __launch_bounds__(256) void kv_join_kernel(const KvAttend a, const Plan p) {
  using T = kv_elem<QT>;
  __shared__ float part[256];
  __shared__ float tops[16], all[16];
  const int tid = threadIdx.x, dim = a.pages.dim;
  Piece u;
  Pieces w;
  int me, joiners;  // which of the unit's workgroups this is, how many may join
  if constexpr (GRID) {
    joiners = gridDim.y;
    const int unit = blockIdx.x;
    u.seq = unit / a.pages.heads;
    u.head = unit - u.seq * a.pages.heads;
    u.len = kv_length(a.lengths, u.seq, a.max_length);
    u.tiles = tiles_of(p, u.len);
    me = blockIdx.y;
    const int chunk = chunk_of(p, u.tiles);
    u.first = me * chunk;
    u.last = min(u.first + chunk, u.tiles);
    w.count = (u.tiles + chunk - 1) / chunk;
    w.head = unit * p.pieces;
    w.next = w.head + 1;
    w.step = 1;
    if (w.count == 1 || me >= w.count) return;
  } else {
    const Slot s = p.slots[blockIdx.x];
    if (!s.valid) return;
    u = s.piece;
    const Shares shares(s.total, p.workgroups);
    const int first = shares.of(s.unit_tile), last = shares.of(s.unit_tile + u.tiles - 1);
    me = (int)blockIdx.x / 2 - first;
    w.count = last - first + 1;
    w.head = 2 * first + (shares.begin(first) == s.unit_tile ? 0 : 1);
    w.next = 2 * (first + 1);
    w.step = 2;
    joiners = w.count;
  }
  for (int qt = 0; qt < p.query_tiles; ++qt) {
    // a run of the output values
    const int rows_here = min(16, p.group - qt * 16), values = rows_here * dim;
    const int n = min(min(w.count, joiners), (values + kJoinValues - 1) / kJoinValues);
    if (!ACC && me >= n) continue;
    total_of(p, w, qt, tops, all);
    const int e0 = me < n ? me * values / n : 0, e1 = me < n ? (me + 1) * values / n : 0;
    const int64_t first_head = (int64_t)u.head * p.group + qt * 16;
    for (int e = e0; e < e1; e += 256) {
      const int width = min(e1 - e, 256), ways = 256 / width;
      const int way = tid / width, mine = e + tid - way * width, q = mine / dim, d = mine - q * dim;
      float o = 0.0f;
      if (way < ways) {
        for (int i0 = way; i0 < w.count; i0 += 4 * ways) {  // four pieces' loads together
          float x[4], m[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int i = i0 + j * ways;
            const int64_t at = (int64_t)w.slot(min(i, w.count - 1)) * p.query_tiles + qt;
            x[j] = p.slot_rows[(at * 16 + q) * DP + d];
            m[j] = i < w.count ? p.slot_ml[at * 32 + q] : -INFINITY;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) o += m[j] == -INFINITY ? 0.0f : x[j] * exp2_of(m[j] - tops[q]);
        }
      }
      __syncthreads();
      part[tid] = o;
      __syncthreads();
      if (way == 0) {
        for (int i = 1; i < ways; ++i) o += part[i * width + tid];
        const float f = all[q] == -INFINITY ? 0.0f : exp2_of(tops[q] - all[q]);
        reinterpret_cast<T*>(a.out)[u.seq * a.out_seq_stride + (first_head + q) * a.out_head_stride + d] = (T)(o * f);
      }
    }
    if (a.lse && me == 0 && tid < rows_here) a.lse[u.seq * (int64_t)a.q_heads + first_head + tid] = all[tid] * kLn2;
    if constexpr (ACC) add_weights(a, p, u, qt, all);
  }
}

// A cache without pages: every sequence is empty.
template <int QT>
__global__ __launch_bounds__(256) void kv_empty_kernel(const KvAttend a) {
  using T = kv_elem<QT>;
  const int64_t s = blockIdx.x;
  for (int i = threadIdx.x; i < a.q_heads * a.pages.dim; i += 256) {
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
  bool grid;
  unsigned units;
  size_t bytes;
};

// Tiles of a grid workgroup, 0: stream mode.  The lengths are not known here, only the tables'
// extent; all figures are for 128 values of 16 bits, 4 queries a key head and 128-slot tiles.
//   Whole units, one launch, up to 4 tiles (one piece 12.2 us, 32 pieces and a join 10.3 us for one
//   sequence of 4,096 slots, but 34.9 against 43.4 us for 256 of 32 to 512), and up to 16 where
//   there are units for all CUs (64 sequences of 125 to 2,000 slots: whole 33.9, pieces of 8 42.3).
//   One sequence: 256 pieces, one a CU, are enough (200,001 slots: 144 us, stream 155, pieces of 16
//   tiles 165; 16,384: 17.7, stream 23.6, 1 tile 22.0). Its tiles are shared by these pieces as its
//   length asks for, which only the kernels know: its table may be far longer.
//   4-bit pages: 768 (200,001 slots of 8 key heads, 64 values: 66 us, 1,024 pieces 59; of one head 41 and 54; 16,000 of
//   8 heads 12.3 and 14.7; 256 values: 93, 512 pieces 89; of one head 51 and 41; 16,000 slots 19 and 19).
//   Several may be much shorter than the longest: smaller pieces (7 of 33 to 30,011 slots, 2 key
//   heads: pieces of 4 tiles 22 us, 8 29, stream 35; 64 of 512 to 8,192: 8 tiles 180, 16 188, stream 186).
//   In f32 (64-slot tiles) 8 is the most: 48 sequences of up to 2,000 slots 30.5 us, 12 32.2.
//   An empty workgroup costs 1.2 ns, so tables far longer than the sequences go to stream mode
//   (64 sequences of up to 2,000 slots in tables of 131,072: stream 41 us, pieces of 12 tiles 91;
//   in tables of 32,768: 42 and 44).
int64_t grid_chunk(int64_t seqs, int64_t units, int64_t tiles, int tile, int ct) {
  const int64_t all = units * tiles, most = tile < 128 ? 8 : 12;
  int64_t chunk = std::min(most, (all + 1023) / 1024);
  if (tiles <= 4 || (tiles <= 16 && units >= 256)) chunk = tiles;
  else if (seqs == 1) chunk = ct == kMXFP4 ? (all + 767) / 768 : (all + 255) / 256;
  const int64_t pieces = (tiles + chunk - 1) / chunk;
  return pieces == 1 || units * pieces <= 8192 ? chunk : 0;
}

constexpr int64_t kFewScores = 32 << 20;  // 128 MiB

Layout layout_of(const KvAttend& a, void* workspace) {
  Layout r{};
  Plan& p = r.plan;
  p.group = a.q_heads / a.pages.heads;
  p.query_tiles = (p.group + 15) / 16;
  p.tile = 4 * step_slots(a.dtype);
  const int64_t tiles = std::max<int64_t>(1, (a.max_length + p.tile - 1) / p.tile);
  const int64_t units = a.seqs * a.pages.heads;
  r.units = (unsigned)units;
  const int dp = padded_dim(a.pages.dim);
  const int64_t chunk = grid_chunk(a.seqs, units, tiles, p.tile, a.pages.dtype);
  r.grid = chunk > 0;
  p.chunk = a.seqs == 1 ? 0 : (int)chunk;
  p.pieces = r.grid ? (int)((tiles + chunk - 1) / chunk) : 0;
  // what the 256 CUs hold at once
  p.workgroups = (int)std::min<int64_t>(256 * waves_per_simd(a.pages.dtype, dp), units * tiles);
  uint8_t* at = static_cast<uint8_t*>(workspace);
  auto take = [&](size_t n) {
    void* x = at + r.bytes;
    r.bytes += (n + 15) / 16 * 16;
    return x;
  };
  const size_t slots = r.grid ? (p.pieces == 1 ? 0 : (size_t)units * p.pieces) : 2 * (size_t)p.workgroups;
  p.slot_rows = static_cast<float*>(take(slots * p.query_tiles * 16 * dp * 4));
  p.slot_ml = static_cast<float*>(take(slots * p.query_tiles * 32 * 4));
  if (!r.grid) p.slots = static_cast<Slot*>(take(slots * sizeof(Slot)));
  if (a.accumulate) {
    // Sequences may be far shorter than their tables: no page belongs to two of them, so scores by
    // slot hold no more than the cache.  In order they are read in longer runs (64 sequences of 512 to
    // 8,192 slots, 32 query heads: 180 us, by slot 187), so that is left where it saves little.
    const int64_t in_order = a.seqs * a.q_heads * tiles * p.tile, of_cache = a.pages.num_pages * a.pages.page * a.q_heads;
    p.by_slot = in_order > kFewScores && in_order > 4 * of_cache;
    p.score_row = p.by_slot ? of_cache / p.group : tiles * p.tile;
    p.scores = static_cast<float*>(take((size_t)(p.by_slot ? of_cache : in_order) * 4));
  }
  return r;
}

template <int QT, int CT, int DP, bool EXACT, bool ACC>
hipError_t launch_kernels(const KvAttend& a, const Layout& l, hipStream_t stream) {
  if (l.grid) {
    const dim3 grid(l.units, (unsigned)l.plan.pieces);
    kv_attend_kernel<QT, CT, DP, EXACT, ACC, true><<<grid, 256, 0, stream>>>(a, l.plan);
    // weights are added piece by piece; to join alone, some workgroups a unit are enough
    const unsigned join = ACC ? grid.y : std::min(grid.y, std::max(1u, 1024 / l.units));
    if (l.plan.pieces > 1) kv_join_kernel<QT, DP, ACC, true><<<dim3(l.units, join), 256, 0, stream>>>(a, l.plan);
  } else {
    const unsigned n = (unsigned)l.plan.workgroups;
    kv_attend_kernel<QT, CT, DP, EXACT, ACC, false><<<n, 256, 0, stream>>>(a, l.plan);
    kv_join_kernel<QT, DP, ACC, false><<<2 * n, 256, 0, stream>>>(a, l.plan);
  }
  return hipGetLastError();
}

template <int QT, int CT, int DP, bool EXACT>
hipError_t launch_dim(const KvAttend& a, const Layout& l, hipStream_t stream) {
  if (a.pages.num_pages == 0) {
    kv_empty_kernel<QT><<<(unsigned)a.seqs, 256, 0, stream>>>(a);
    return hipGetLastError();
  }
  return a.accumulate ? launch_kernels<QT, CT, DP, EXACT, true>(a, l, stream)
                      : launch_kernels<QT, CT, DP, EXACT, false>(a, l, stream);
}

template <int QT, int CT>
hipError_t launch_types(const KvAttend& a, void* workspace, hipStream_t stream) {
  const Layout l = layout_of(a, workspace);
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

}  // namespace nve_amd
