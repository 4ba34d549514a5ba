// kv_evict.hip -- eviction from the paged key-value cache by accumulated
// attention weight.
//
// kv_select_kernel, one workgroup per (sequence, key head): the n = length -
// budget slots to drop are the first in (protected, key, slot), key being the
// weight's bits in an order-preserving form.  If there are at most n
// unprotected slots all of them go, and the rest is found among the protected
// ones; otherwise it is found among the unprotected.  A radix select, eight
// bits a pass, gives the key T of the last one dropped and how many slots of
// that very key go (the first ones).  Two ordered scans over the slots then
// list the dropped slots below the budget and pair the kept ones past it with
// them.  kv_move_kernel copies the rows of the pairs.  No pair's source is
// another's target (sources lie past the budget, targets below it), so the
// copies need no order.
#include "kv_common.cuh"

namespace nve_amd {

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kMoveThreads = 256;

// Ascending order of the keys is that of the weights: -infinity first, NaN
// last, the two zeros equal.
__device__ __forceinline__ uint32_t order_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t b = __float_as_uint(w + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct Slot {
  uint32_t key;
  bool held;  // protected
};

struct Head {
  KvPages pages;
  const int32_t* table;
  int head;
  int64_t newest, sinks, recent;

  __device__ __forceinline__ Slot slot(int64_t t) const {
    const int64_t page = kv_page(pages, table, t);
    if (page < 0) return {0u, false};  // absent: below every weight's key
    const int64_t at = kv_row(pages, page, head, t);
    const int64_t i = pages.index[at];
    return {order_key(pages.weights[at]), i < sinks || i > newest - recent};
  }
};

__device__ __forceinline__ int64_t block_max(int64_t v, int64_t* red) {
  for (int m = 32; m > 0; m >>= 1) {
    const int64_t o = __shfl_xor(v, m);
    v = o > v ? o : v;
  }
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < kWaves; ++w) v = red[w] > v ? red[w] : v;
  __syncthreads();
  return v;
}

__device__ __forceinline__ int block_count(bool on, int* red) {
  const int n = __popcll(__ballot(on));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = n;
  __syncthreads();
  int sum = 0;
  for (int w = 0; w < kWaves; ++w) sum += red[w];
  __syncthreads();
  return sum;
}

// How many threads before this one have `on`; *total: how many in the workgroup.
__device__ __forceinline__ int block_rank(bool on, int* red, int* total) {
  const uint64_t bits = __ballot(on);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (lane == 0) red[wave] = __popcll(bits);
  __syncthreads();
  int before = 0, sum = 0;
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) before += red[w];
    sum += red[w];
  }
  __syncthreads();
  *total = sum;
  return before + __popcll(bits & ((1ull << lane) - 1));
}

// Pairs of a (sequence, head): row numbers to[] and from[], `counts` of them.
__global__ __launch_bounds__(kThreads) void kv_select_kernel(const KvEvict a, int64_t* to, int64_t* from,
                                                             int32_t* counts, int64_t max_pairs) {
  __shared__ int64_t red64[kWaves];
  __shared__ int red[kWaves];
  __shared__ int hist[256];
  __shared__ int chosen[2];
  const int tid = threadIdx.x;
  const int64_t s = blockIdx.x;
  const int head = blockIdx.y;
  const int64_t unit = s * a.pages.heads + head;
  const int64_t len = kv_length(a.lengths, s, a.max_length);
  const int64_t keep = len < a.budget ? len : a.budget;
  if (head == 0 && tid == 0) a.new_lengths[s] = (int32_t)keep;
  const int64_t drop = len - keep;
  if (tid == 0) counts[unit] = 0;
  if (drop == 0 || keep == 0) return;
  Head h{a.pages, a.tables + s * a.table_stride, head, 0, a.sinks, a.recent};

  int64_t newest = INT64_MIN / 2;
  for (int64_t t = tid; t < len; t += kThreads) {
    const int64_t page = kv_page(a.pages, h.table, t);
    if (page < 0) continue;
    const int64_t i = a.pages.index[kv_row(a.pages, page, head, t)];
    newest = i > newest ? i : newest;
  }
  h.newest = block_max(newest, red64);
  int64_t open = 0;  // unprotected slots
  for (int64_t t0 = 0; t0 < len; t0 += kThreads) open += block_count(t0 + tid < len && !h.slot(t0 + tid).held, red);
  const bool among_held = drop > open;       // every unprotected slot goes, and some protected ones
  int rest = (int)(among_held ? drop - open : drop);  // how many of the class go
  uint32_t prefix = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int64_t t = tid; t < len; t += kThreads) {
      const Slot x = h.slot(t);
      if (x.held == among_held && (shift == 24 || (x.key >> (shift + 8)) == (prefix >> (shift + 8))))
        atomicAdd(&hist[(x.key >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {  // the digit of the rest-th one
      int n = rest, d = 0;
      while (d < 255 && n > hist[d]) n -= hist[d++];
      chosen[0] = d;
      chosen[1] = n;
    }
    __syncthreads();
    prefix |= (uint32_t)chosen[0] << shift;
    rest = chosen[1];
    __syncthreads();
  }

  // rest slots of key `prefix` go, the first ones
  int equal = 0, holes = 0, movers = 0;
  for (int64_t t0 = 0; t0 < len; t0 += kThreads) {
    const int64_t t = t0 + tid;
    const bool in = t < len;
    const Slot x = in ? h.slot(t) : Slot{0u, false};
    const bool same = in && x.held == among_held && x.key == prefix;
    int n;
    const int rank = equal + block_rank(same, red, &n);
    equal += n;
    const bool dropped = x.held != among_held ? !x.held : x.key < prefix || (same && rank < rest);
    const bool hole = in && dropped && t < keep;
    const bool mover = in && !dropped && t >= keep;
    const int hr = holes + block_rank(hole, red, &n);
    holes += n;
    const int mr = movers + block_rank(mover, red, &n);
    movers += n;
    if (hole || mover) {
      const int64_t page = kv_page(a.pages, h.table, t);
      (hole ? to : from)[unit * max_pairs + (hole ? hr : mr)] = page < 0 ? -1 : kv_row(a.pages, page, head, t);
    }
  }
  if (tid == 0) counts[unit] = holes;
}

// One row a wave at a time.
__global__ __launch_bounds__(kMoveThreads) void kv_move_kernel(const KvEvict a, const int64_t* to, const int64_t* from,
                                                               const int32_t* counts, int64_t max_pairs) {
  const int64_t unit = blockIdx.x;
  const int lane = threadIdx.x & 63;
  const int waves = (int)gridDim.y * (kMoveThreads / 64);
  const int n = counts[unit];
  const KvPages& c = a.pages;
  const int words = c.dim * value_elem_bytes(c.dtype) / 8;  // head_dim is a multiple of 8
  for (int i = (int)blockIdx.y * (kMoveThreads / 64) + (threadIdx.x >> 6); i < n; i += waves) {
    const int64_t dst = to[unit * max_pairs + i], src = from[unit * max_pairs + i];
    if (dst < 0 || src < 0) continue;
    for (int w = lane; w < words; w += 64) {
      reinterpret_cast<uint64_t*>(c.k)[dst * words + w] = reinterpret_cast<const uint64_t*>(c.k)[src * words + w];
      reinterpret_cast<uint64_t*>(c.v)[dst * words + w] = reinterpret_cast<const uint64_t*>(c.v)[src * words + w];
    }
    if (lane == 0) {
      c.weights[dst] = c.weights[src];
      c.index[dst] = c.index[src];
      if (c.k_scale) {
        c.k_scale[dst] = c.k_scale[src];
        c.v_scale[dst] = c.v_scale[src];
      }
    }
  }
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
  kv_select_kernel<<<dim3((unsigned)a.seqs, (unsigned)a.pages.heads), kThreads, 0, stream>>>(a, to, from, counts,
                                                                                            pairs);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || pairs == 0) return e;
  const int64_t rows = (pairs + 3) / 4;
  kv_move_kernel<<<dim3((unsigned)units, (unsigned)(rows < 64 ? rows : 64)), kMoveThreads, 0, stream>>>(
      a, to, from, counts, pairs);
  return hipGetLastError();
}

}  // namespace nve_amd
