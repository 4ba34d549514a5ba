// kv_evict.hip -- eviction from the paged key-value cache by accumulated
// attention weight.
//
// kv_select_kernel, one workgroup per (sequence, key head): the n = length -
// budget slots to drop are the first in (protected, key, slot), key being the
// weight's bits in an order-preserving form.  If there are at most n
// unprotected slots all of them go, and the rest is found among the protected
// ones; otherwise it is found among the unprotected.  A radix select of 11, 11
// and 10 bits gives the key T of the last one dropped and how many slots of
// that very key go (the first ones).  A scan over the slots then numbers the
// dropped ones below the budget and the kept ones past it, which are paired in
// order.  No pair's source is another's target (sources lie past the budget,
// targets below it), so the rows of the pairs are copied in any order: by the
// workgroup itself where there can be only a few, else by kv_move_kernel.
//
// Bound: for short tables the chain of dependent steps (page number, weight,
// three histograms, two scans), else the bytes of the moved rows.  A thread has
// consecutive slots, 4 at a time as they lie in a page, and keeps their keys in
// registers up to kRegister slots a thread; longer sequences read the weights
// again in every pass.  11 bits a digit, because weights that fall off over some
// binades share their first 8 bits: their additions to one bin would queue.
#include <algorithm>

#include "kv_common.cuh"

namespace nve_amd {

namespace {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using i32x4 = __attribute__((ext_vector_type(4))) int32_t;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;

constexpr int kBins = 2048;
constexpr int64_t kFewPairs = 64;  // of a unit: copied by the selecting workgroup

// Ascending order of the keys is that of the weights: -infinity first, NaN
// last, the two zeros equal.
__device__ __forceinline__ uint32_t order_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t b = __float_as_uint(w + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Sums of two counts over the threads before this one, and over all.
template <int THREADS>
struct Scan {
  static constexpr int kWaves = THREADS / 64;
  int before[2], total[2];
  __device__ __forceinline__ Scan(int a, int b, int (*red)[2]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = a, y = b;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int ox = __shfl_up(x, d), oy = __shfl_up(y, d);
      if (lane >= d) {
        x += ox;
        y += oy;
      }
    }
    __syncthreads();
    if (lane == 63) {
      red[wave][0] = x;
      red[wave][1] = y;
    }
    __syncthreads();
    before[0] = x - a;
    before[1] = y - b;
    total[0] = total[1] = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) {
        before[0] += red[w][0];
        before[1] += red[w][1];
      }
      total[0] += red[w][0];
      total[1] += red[w][1];
    }
  }
};

// A word of 16 or 8 bytes of a k row and of its v row; word 0 brings what goes with the row.
template <typename WORD>
struct Moved {
  WORD k, v;
  float weight, k_scale, v_scale;
  int32_t place;
  __device__ __forceinline__ void load(const KvPages& c, int64_t row, int words, int word) {
    k = reinterpret_cast<const WORD*>(c.k)[row * words + word];
    v = reinterpret_cast<const WORD*>(c.v)[row * words + word];
    if (word == 0) {
      weight = c.weights[row];
      place = c.index[row];
      if (c.k_scale) {
        k_scale = c.k_scale[row];
        v_scale = c.v_scale[row];
      }
    }
  }
  __device__ __forceinline__ void store(const KvPages& c, int64_t row, int words, int word) const {
    reinterpret_cast<WORD*>(c.k)[row * words + word] = k;
    reinterpret_cast<WORD*>(c.v)[row * words + word] = v;
    if (word == 0) {
      c.weights[row] = weight;
      c.index[row] = place;
      if (c.k_scale) {
        c.k_scale[row] = k_scale;
        c.v_scale[row] = v_scale;
      }
    }
  }
};

// Words first, first + step, .. of `count` pairs' rows: AHEAD of them are loaded, then stored.
template <typename WORD, int AHEAD>
__device__ __forceinline__ void move_rows(const KvPages& c, const int64_t* to, const int64_t* from, int count,
                                          int64_t first, int64_t step) {
  const int words = c.dim * value_elem_bytes(c.dtype) / (int)sizeof(WORD);
  const int64_t n = (int64_t)count * words;
  for (int64_t e0 = first; e0 < n; e0 += AHEAD * step) {
    Moved<WORD> x[AHEAD];
    int64_t dst[AHEAD], src[AHEAD];
    int word[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int64_t e = e0 + j * step;
      const int64_t i = n <= UINT32_MAX ? (int64_t)((uint32_t)e / (uint32_t)words) : e / words;
      word[j] = (int)(e - i * words);
      dst[j] = e < n ? to[i] : -1;
      src[j] = e < n ? from[i] : -1;
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (dst[j] >= 0 && src[j] >= 0) x[j].load(c, src[j], words, word[j]);  // else a row of an absent page
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (dst[j] >= 0 && src[j] >= 0) x[j].store(c, dst[j], words, word[j]);
  }
}

template <int AHEAD>
__device__ __forceinline__ void move_rows(const KvPages& c, const int64_t* to, const int64_t* from, int count,
                                          int64_t first, int64_t step) {
  if (c.dim * value_elem_bytes(c.dtype) % 16 == 0) move_rows<u32x4, AHEAD>(c, to, from, count, first, step);
  else move_rows<uint64_t, AHEAD>(c, to, from, count, first, step);
}

// PER: slots of a thread that are kept in registers, 0: none.
template <int THREADS, int PER>
__global__ __launch_bounds__(THREADS) void kv_select_kernel(const KvEvict a, int64_t* to, int64_t* from,
                                                            int32_t* counts, int64_t max_pairs, int few) {
  constexpr int kWaves = THREADS / 64, kRegs = PER > 0 ? PER : 4;
  __shared__ int hist[kBins];
  __shared__ int red[kWaves][2];
  __shared__ int chosen[2];
  const int tid = threadIdx.x;
  const int64_t s = blockIdx.x;
  const int head = blockIdx.y;
  const int64_t unit = s * a.pages.heads + head;
  const int len = (int)kv_length(a.lengths, s, a.max_length);
  const int keep = len < a.budget ? len : (int)a.budget;
  if (head == 0 && tid == 0) a.new_lengths[s] = keep;
  const int drop = len - keep;
  if (drop == 0 || keep == 0) {
    if (tid == 0) counts[unit] = 0;
    return;
  }
  const int32_t* table = a.tables + s * a.table_stride;
  const int per = PER > 0 ? PER : ((len + THREADS - 1) / THREADS + 3) / 4 * 4;
  const int t0 = min(tid * (int64_t)per, (int64_t)len), t1 = min(t0 + per, len);

  // Four slots: their keys and places; those of an absent page come first of all and are not protected.
  struct Four {
    uint32_t key[4];
    int place[4];
    bool there;
  };
  auto read = [&](int t) {
    Four f;
    const int64_t page = kv_page(a.pages, table, t);
    f.there = page >= 0;
    f32x4 w = {0.0f, 0.0f, 0.0f, 0.0f};
    i32x4 i = {0, 0, 0, 0};
    if (f.there) {
      typedef f32x4 __attribute__((aligned(4))) f4;
      typedef i32x4 __attribute__((aligned(4))) i4;
      const int64_t at = kv_row(a.pages, page, head, t);
      w = *reinterpret_cast<const f4*>(a.pages.weights + at);
      i = *reinterpret_cast<const i4*>(a.pages.index + at);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f.key[j] = f.there ? order_key(w[j]) : 0u;
      f.place[j] = i[j];
    }
    return f;
  };

  // the newest place, and the keys
  uint32_t key[kRegs];
  int place[kRegs];
  uint32_t there = 0;  // a bit per four slots
  int newest = INT32_MIN;
  if constexpr (PER > 0) {
#pragma unroll
    for (int j = 0; j < PER; j += 4) {
      Four f{};
      if (t0 + j < t1) f = read(t0 + j);
      if (f.there) there |= 1u << (j / 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        key[j + i] = f.key[i];
        place[j + i] = f.place[i];
        if (f.there && t0 + j + i < t1) newest = max(newest, f.place[i]);
      }
    }
  } else {
    for (int t = t0; t < t1; t += 4) {
      const Four f = read(t);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (f.there && t + i < t1) newest = max(newest, f.place[i]);
    }
  }
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) newest = max(newest, __shfl_xor(newest, m));
  if ((tid & 63) == 0) red[tid >> 6][0] = newest;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) newest = max(newest, red[w][0]);
  // places above `line` are protected, those below a.sinks too
  const int64_t line = (int64_t)newest - a.recent;
  auto protects = [&](int place) { return place < a.sinks || place > line; };

  // every slot of this thread: f(slot, key, protected)
  uint32_t held = 0;
  auto each = [&](auto f) {
    if constexpr (PER > 0) {
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (t0 + j < t1) f(t0 + j, key[j], (bool)((held >> j) & 1));
    } else {
      for (int t = t0; t < t1; t += 4) {
        const Four x = read(t);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (t + i < t1) f(t + i, x.key[i], x.there && protects(x.place[i]));
      }
    }
  };
  int open = 0;  // unprotected slots
  if constexpr (PER > 0) {
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (((there >> (j / 4)) & 1) && protects(place[j])) held |= 1u << j;
  }
  each([&](int, uint32_t, bool h) { open += h ? 0 : 1; });
  open = Scan<THREADS>(open, 0, red).total[0];
  const bool among_held = drop > open;           // every unprotected slot goes, and some protected ones
  int rest = among_held ? drop - open : drop;    // how many of the class go
  uint32_t prefix = 0, above = 0;                // the digits found so far, and their bits
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    constexpr int kOwn = kBins / THREADS;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) hist[tid * kOwn + i] = 0;
    __syncthreads();
    each([&](int, uint32_t k, bool h) {
      if (h == among_held && (k & above) == prefix) atomicAdd(&hist[(k >> shift) & ((1 << bits) - 1)], 1);
    });
    __syncthreads();
    // the digit of the rest-th one
    int own[kOwn], sum = 0;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) sum += own[i] = hist[tid * kOwn + i];
    int before = Scan<THREADS>(sum, 0, red).before[0];
    if (before < rest && rest <= before + sum) {
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        if (before < rest && rest <= before + own[i]) {
          chosen[0] = tid * kOwn + i;
          chosen[1] = rest - before;
        }
        before += own[i];
      }
    }
    __syncthreads();
    prefix |= (uint32_t)chosen[0] << shift;
    above |= ((1u << bits) - 1) << shift;
    rest = chosen[1];
  }

  // `rest` slots of key `prefix` go, the first ones
  int same = 0;
  each([&](int, uint32_t k, bool h) { same += h == among_held && k == prefix ? 1 : 0; });
  const int same_before = Scan<THREADS>(same, 0, red).before[0];
  auto drops = [&](uint32_t k, bool h, int& seen) {
    if (h != among_held) return !h;
    if (k != prefix) return k < prefix;
    return seen++ < rest;
  };
  int holes = 0, movers = 0, seen = same_before;
  each([&](int t, uint32_t k, bool h) {
    const bool d = drops(k, h, seen);
    if (t < keep) holes += d ? 1 : 0;
    else movers += d ? 0 : 1;
  });
  const Scan<THREADS> scan(holes, movers, red);
  int hole = scan.before[0], mover = scan.before[1];
  seen = same_before;
  each([&](int t, uint32_t k, bool h) {
    const bool d = drops(k, h, seen);
    if (d != (t < keep)) return;
    const int64_t page = kv_page(a.pages, table, t);
    const int64_t row = page < 0 ? -1 : kv_row(a.pages, page, head, t);
    if (d) to[unit * max_pairs + hole++] = row;
    else from[unit * max_pairs + mover++] = row;
  });
  const int count = scan.total[0];
  if (tid == 0) counts[unit] = count;
  if (!few) return;
  __threadfence_block();  // the pairs
  __syncthreads();
  move_rows<1>(a.pages, to + unit * max_pairs, from + unit * max_pairs, count, tid, THREADS);
}

constexpr int kMoveThreads = 256;
constexpr int kMoveAhead = 4;

__global__ __launch_bounds__(kMoveThreads) void kv_move_kernel(const KvEvict a, const int64_t* to, const int64_t* from,
                                                               const int32_t* counts, int64_t max_pairs) {
  const int64_t unit = blockIdx.x;
  move_rows<kMoveAhead>(a.pages, to + unit * max_pairs, from + unit * max_pairs, counts[unit],
                        (int64_t)blockIdx.y * kMoveThreads + threadIdx.x, (int64_t)gridDim.y * kMoveThreads);
}

// A unit's pairs: no more than slots are kept, or are dropped.
int64_t max_pairs(const KvEvict& a) {
  const int64_t drop = a.max_length > a.budget ? a.max_length - a.budget : 0;
  return drop < a.budget ? drop : a.budget;
}

}  // namespace

size_t kv_evict_workspace(const KvEvict& a) {
  const size_t units = (size_t)a.seqs * (size_t)a.pages.heads;
  return units * (size_t)max_pairs(a) * 16 + (units * 4 + 15) / 16 * 16;
}

hipError_t launch_kv_evict(const KvEvict& a, void* workspace, hipStream_t stream) {
  if (a.seqs == 0) return hipSuccess;
  const int64_t units = a.seqs * a.pages.heads, pairs = max_pairs(a);
  int64_t* to = static_cast<int64_t*>(workspace);
  int64_t* from = to + units * pairs;
  int32_t* counts = reinterpret_cast<int32_t*>(from + units * pairs);
  const int few = pairs <= kFewPairs;
  const dim3 grid((unsigned)a.seqs, (unsigned)a.pages.heads);
  if (a.max_length <= 1024)
    kv_select_kernel<256, 4><<<grid, 256, 0, stream>>>(a, to, from, counts, pairs, few);
  else if (a.max_length <= 4096)
    kv_select_kernel<256, 16><<<grid, 256, 0, stream>>>(a, to, from, counts, pairs, few);
  else if (a.max_length <= 16384)
    kv_select_kernel<1024, 16><<<grid, 1024, 0, stream>>>(a, to, from, counts, pairs, few);
  else if (a.max_length <= 32768)
    kv_select_kernel<1024, 32><<<grid, 1024, 0, stream>>>(a, to, from, counts, pairs, few);
  else
    kv_select_kernel<1024, 0><<<grid, 1024, 0, stream>>>(a, to, from, counts, pairs, few);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || few) return e;
  // enough workgroups to fill the machine, each with some rounds of its words
  const int64_t words = pairs * a.pages.dim * value_elem_bytes(a.pages.dtype) / 8;
  const int64_t most = std::max<int64_t>(1, 16384 / units);
  const int64_t y = std::min(most, (words + kMoveThreads * kMoveAhead - 1) / (kMoveThreads * kMoveAhead));
  kv_move_kernel<<<dim3((unsigned)units, (unsigned)std::max<int64_t>(1, y)), kMoveThreads, 0, stream>>>(a, to, from,
                                                                                                     counts, pairs);
  return hipGetLastError();
}

}  // namespace nve_amd
