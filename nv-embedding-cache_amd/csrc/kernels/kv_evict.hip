// kv_evict.hip -- eviction from the paged key-value cache by accumulated
// attention weight.
//
// kv_select_kernel, one workgroup per (sequence, key head): the n = length -
// budget slots to drop are the first in (protected, weight, slot).  Weights
// become keys of the same order.  If there are at most n unprotected slots, all
// of them go: their keys become the lowest; otherwise no protected one goes:
// theirs become the highest.  A radix select of 11, 11 and 10 bits then finds
// the key of the n-th slot and how many slots of that very key go (the first
// ones), and stops early once all that share the bits found so far go.  A scan
// over the slots in order numbers the dropped ones below the budget and the kept
// ones past it, which are paired.  No pair's source is another's target (sources
// lie past the budget, targets below it), so the rows of the pairs are copied in
// any order: by the workgroup itself where there can be only a few, else by
// kv_move_kernel.
//
// Bound: for short tables the chain of dependent steps (page number, weight, two
// or three histograms, a scan), else the bytes of the moved rows.  A thread reads
// four slots at a time, as they lie in a page, neighbours next to each other, and
// keeps their keys in registers; sequences longer than those hold read them again
// in every pass.  For the scan each slot's class (goes, equal, stays) passes
// through shared memory in two bits, so that a thread has slots in a row.  11 bits
// a digit, because weights that fall off over some binades share their first 8
// bits: their additions to one bin would queue.
// Measured: 64 sequences of 2,064 slots and 8 key heads to 2,048: 15 us
// repeated on one cache, 16 to 19 on a fresh one; 8 prompts of 32,768 slots to 4,096: 41
// to 44 us to choose (64 workgroups on 256 CUs) and 58 to 74 to move the rows of a fresh
// cache, 35 and 9 once repeated, as fewer rows then move.
#include <algorithm>
#include <type_traits>

#include "kv_common.cuh"

namespace nve_amd {

namespace {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using i32x4 = __attribute__((ext_vector_type(4))) int32_t;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;

constexpr int kBins = 2048;
// Pairs of a unit that the selecting workgroup copies itself.  One launch / two, us a call on fresh
// caches, 8 key heads of 128 bf16 values: 64 sequences of 2,000 slots, 64 pairs 19.2 / 22.3, 256 pairs
// 34.8 / 36.0, 512 59.2 / 56.0; 8 sequences 14.4 / 17.7, 128 pairs 17.6 / 18.5, 256 20.6 / 18.6.
constexpr int64_t kFewPairs = 64;

// Ascending order of the keys is that of the weights: -infinity first, NaN
// last, the two zeros equal.  No weight has one of the keys below.
constexpr uint32_t kGoes = 0u;           // dropped in any case
constexpr uint32_t kAbsent = 1u;         // of an absent page: before every weight
constexpr uint32_t kNaN = 0xffc00000u;   // past +infinity's 0xff800000
constexpr uint32_t kStays = 0xffffffffu; // kept in any case, or no slot
// The select may end after the first 11 bits, and neither slots that stay nor slots that go are
// counted in it: no key that is counted beside them may share those bits.  Beside slots that go
// these are protected slots' only, whose pages are there (from -infinity's 0x007fffff on).
constexpr int kFirstShift = 21;
static_assert(kNaN >> kFirstShift != kStays >> kFirstShift && 0x007fffffu >> kFirstShift != kGoes >> kFirstShift);
__device__ __forceinline__ uint32_t order_key(float w) {
  const uint32_t b = __float_as_uint(w + 0.0f);
  return w != w ? kNaN : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

// Sums of N counts over the threads before this one, and over all.
template <int THREADS, int N>
struct Scan {
  static constexpr int kWaves = THREADS / 64;
  static_assert(kWaves % 4 == 0);
  int before[N], total[N];
  __device__ __forceinline__ Scan(const int (&x)[N], int (*red)[kWaves]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int sum[N];
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] = wave_scan(x[i]);
    __syncthreads();
    if (lane == 63) {
#pragma unroll
      for (int i = 0; i < N; ++i) red[i][wave] = sum[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      before[i] = sum[i] - x[i];
      total[i] = 0;
#pragma unroll
      for (int w = 0; w < kWaves; w += 4) {
        const i32x4 r = *reinterpret_cast<const i32x4*>(&red[i][w]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          before[i] += w + j < wave ? r[j] : 0;
          total[i] += r[j];
        }
      }
    }
  }
};

// A word of 16 or 8 bytes of a k row and of its v row; word 0 brings what goes with the row.  A
// kMXFP4 row has as many scales (bytes) as words of 16 bytes: each word brings one.
template <typename WORD>
struct Moved {
  WORD k, v;
  float weight;
  uint32_t k_scale, v_scale;
  int32_t place;
  __device__ __forceinline__ void load(const KvPages& c, int64_t row, int words, int word) {
    k = reinterpret_cast<const WORD*>(c.k)[row * words + word];
    v = reinterpret_cast<const WORD*>(c.v)[row * words + word];
    if (c.dtype == kMXFP4) {
      k_scale = static_cast<const uint8_t*>(c.k_scale)[row * words + word];
      v_scale = static_cast<const uint8_t*>(c.v_scale)[row * words + word];
    }
    if (word == 0) {
      weight = c.weights[row];
      place = c.index[row];
      if (c.dtype == kE4M3) {
        k_scale = static_cast<const uint32_t*>(c.k_scale)[row];
        v_scale = static_cast<const uint32_t*>(c.v_scale)[row];
      }
    }
  }
  __device__ __forceinline__ void store(const KvPages& c, int64_t row, int words, int word) const {
    reinterpret_cast<WORD*>(c.k)[row * words + word] = k;
    reinterpret_cast<WORD*>(c.v)[row * words + word] = v;
    if (c.dtype == kMXFP4) {
      static_cast<uint8_t*>(c.k_scale)[row * words + word] = (uint8_t)k_scale;
      static_cast<uint8_t*>(c.v_scale)[row * words + word] = (uint8_t)v_scale;
    }
    if (word == 0) {
      c.weights[row] = weight;
      c.index[row] = place;
      if (c.dtype == kE4M3) {
        static_cast<uint32_t*>(c.k_scale)[row] = k_scale;
        static_cast<uint32_t*>(c.v_scale)[row] = v_scale;
      }
    }
  }
};

constexpr int kPairs = 64;  // resolved at a time

// Pairs first .. last - 1 of a head's lists (slots): their rows are found first, one pair a
// thread, then all threads copy words, AHEAD of them loaded before they are stored.
template <typename WORD, int THREADS, int AHEAD>
__device__ __forceinline__ void move_words(const KvPages& c, const int32_t* table, int head, const int32_t* to,
                                           const int32_t* from, int64_t first, int64_t last, int64_t (*rows)[2]) {
  const int words = kv_row_bytes(c.dtype, c.dim) / (int)sizeof(WORD);
  for (int64_t p0 = first; p0 < last; p0 += kPairs) {
    const int n = (int)min((int64_t)kPairs, last - p0);
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * n; i += THREADS) {
      const int t = i & 1 ? from[p0 + i / 2] : to[p0 + i / 2];
      const int64_t page = kv_page(c, table, t);
      rows[i / 2][i & 1] = page < 0 ? -1 : kv_row(c, page, head, t);
    }
    __syncthreads();
    for (int e0 = threadIdx.x; e0 < n * words; e0 += AHEAD * THREADS) {
      Moved<WORD> x[AHEAD];
      int64_t dst[AHEAD], src[AHEAD];
      int word[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int e = e0 + j * THREADS, i = min(e, n * words - 1) / words;
        word[j] = min(e, n * words - 1) - i * words;
        dst[j] = e < n * words ? rows[i][0] : -1;
        src[j] = rows[i][1];
      }
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
        if (dst[j] >= 0 && src[j] >= 0) x[j].load(c, src[j], words, word[j]);  // not of an absent page
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
        if (dst[j] >= 0 && src[j] >= 0) x[j].store(c, dst[j], words, word[j]);
    }
  }
}

template <int THREADS, int AHEAD>
__device__ __forceinline__ void move_rows(const KvPages& c, const int32_t* table, int head, const int32_t* to,
                                          const int32_t* from, int64_t first, int64_t last, int64_t (*rows)[2]) {
  if (kv_row_bytes(c.dtype, c.dim) % 16 == 0)
    move_words<u32x4, THREADS, AHEAD>(c, table, head, to, from, first, last, rows);
  else
    move_words<uint64_t, THREADS, AHEAD>(c, table, head, to, from, first, last, rows);
}

// PER: slots of a thread that are kept in registers, 0: none.
template <int THREADS, int PER>
__global__ __launch_bounds__(THREADS) void kv_select_kernel(const KvEvict a, int32_t* to, int32_t* from,
                                                            int32_t* counts, int64_t max_pairs, int few) {
  constexpr int kWaves = THREADS / 64, kOwn = kBins / THREADS;
  constexpr int kRun = PER == 0 || PER > 32 ? 32 : PER;  // slots of a thread in a round of the ordered scan
  constexpr int kFours = (PER > 0 ? PER : 4) / 4;        // and of four neighbours each, before
  constexpr int kKeys = 4 * kFours;
  using Codes = std::conditional_t<kRun == 32, uint64_t, std::conditional_t<kRun == 16, uint32_t, uint8_t>>;
  static_assert(sizeof(Codes) == kRun / 4);
  __shared__ alignas(16) int hist[kBins];
  __shared__ alignas(8) uint8_t codes[THREADS * kRun / 4];  // two bits a slot
  __shared__ alignas(16) int red[4][kWaves];
  __shared__ int chosen[3];
  __shared__ int32_t few_to[kFewPairs], few_from[kFewPairs];
  __shared__ int64_t few_rows[kPairs][2];
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
  const int fours = len / 4 + (len % 4 != 0);

  // Four slots at a time: their page (-1: absent), places (INT32_MIN where there is no slot)
  // and keys.  Without branches, so that a thread's loads go out together: slots past the
  // length read the last one's.
  auto page_of = [&](int64_t four) {
    const int id = table[4 * min(four, (int64_t)fours - 1) >> a.pages.page_bits];
    return id >= 0 && id < a.pages.num_pages ? id : -1;
  };
  auto at_of = [&](int64_t four, int page) {
    return kv_row(a.pages, max(page, 0), head, 4 * min(four, (int64_t)fours - 1));
  };
  const bool stored = a.pages.num_pages > 0;
  auto read_places = [&](int64_t four, int page, int* place) {
    typedef i32x4 __attribute__((aligned(4))) i4;
    i32x4 i = {0, 0, 0, 0};
    if (stored) i = *reinterpret_cast<const i4*>(a.pages.index + at_of(four, page));
#pragma unroll
    for (int j = 0; j < 4; ++j) place[j] = ((4 * four + j < len) & (page >= 0)) ? i[j] : INT32_MIN;
  };
  auto read_keys = [&](int64_t four, int page, uint32_t* key) {
    typedef f32x4 __attribute__((aligned(4))) f4;
    f32x4 w = {0.0f, 0.0f, 0.0f, 0.0f};
    if (stored) w = *reinterpret_cast<const f4*>(a.pages.weights + at_of(four, page));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t k = page >= 0 ? order_key(w[j]) : kAbsent;
      key[j] = 4 * four + j < len ? k : kStays;
    }
  };

  // the newest place
  int pages[kFours];
  int place[kKeys];
  int newest = INT32_MIN;
  if constexpr (PER > 0) {
#pragma unroll
    for (int r = 0; r < kFours; ++r) pages[r] = page_of(r * THREADS + tid);
#pragma unroll
    for (int r = 0; r < kFours; ++r) read_places(r * THREADS + tid, pages[r], &place[4 * r]);
#pragma unroll
    for (int j = 0; j < PER; ++j) newest = max(newest, place[j]);
  } else {
    for (int64_t q = tid; q < fours; q += THREADS) {
      read_places(q, page_of(q), place);
#pragma unroll
      for (int i = 0; i < 4; ++i) newest = max(newest, place[i]);
    }
  }
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) newest = max(newest, __shfl_xor(newest, m));
  if ((tid & 63) == 0) red[0][tid >> 6] = newest;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) newest = max(newest, red[0][w]);
  // protected: places up to `low` (sinks), and from `high` on (recent); never a slot of an absent page
  const int low = (int)min(a.sinks - 1, (int64_t)INT32_MAX);
  const int high = (int)max((int64_t)newest - a.recent + 1, (int64_t)INT32_MIN);
  const bool any_recent = a.recent > 0;
  auto protects = [&](int place) { return (place <= low) | (any_recent & (place >= high)); };

  // Slots that are protected (a bit per slot in registers), and how many are not.
  int open[1] = {0};
  uint64_t held = 0;
  if constexpr (PER > 0) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int64_t four = (j / 4) * THREADS + tid;
      const bool h = protects(place[j]) & (pages[j / 4] >= 0), in = 4 * four + j % 4 < len;
      held |= h ? 1ull << j : 0ull;
      open[0] += (in & !h) ? 1 : 0;
    }
  } else {
    for (int64_t q = tid; q < fours; q += THREADS) {
      const int page = page_of(q);
      read_places(q, page, place);
#pragma unroll
      for (int i = 0; i < 4; ++i) open[0] += ((4 * q + i < len) & !(protects(place[i]) & (page >= 0))) ? 1 : 0;
    }
  }
  const int opened = Scan<THREADS, 1>(open, red).total[0];
  // Among the protected: every unprotected slot goes, and some protected ones; else no protected one does.
  const bool among_held = drop > opened;
  auto in_order = [&](uint32_t k, bool h) {
    const uint32_t x = among_held ? (h ? k : kGoes) : (h ? kStays : k);
    return k == kStays ? kStays : x;
  };
  uint32_t key[kKeys];
  auto keys_of = [&](int64_t q, uint32_t* k) {  // where they are not in registers
    const int page = page_of(q);
    read_places(q, page, place);
    read_keys(q, page, k);
#pragma unroll
    for (int i = 0; i < 4; ++i) k[i] = in_order(k[i], protects(place[i]) & (page >= 0));
  };
  if constexpr (PER > 0) {
#pragma unroll
    for (int r = 0; r < kFours; ++r) read_keys(r * THREADS + tid, pages[r], &key[4 * r]);
#pragma unroll
    for (int j = 0; j < PER; ++j) key[j] = in_order(key[j], (held >> j) & 1);
  }

  // The digits found so far and their bits: keys below `prefix` in those bits go, and the first
  // `rest` of those equal to it (all of them once as many are left as go).  Slots that go or stay
  // in any case are not counted; no key that is counted has their first digit.
  int rest = among_held ? drop - opened : drop;
  uint32_t prefix = 0, found = 0;
  for (int shift = kFirstShift, bits = 11;;) {
#pragma unroll
    for (int i = 0; i < kOwn; ++i) hist[tid + i * THREADS] = 0;
    __syncthreads();
    const uint32_t digit = (1u << bits) - 1;
    auto count = [&](uint32_t k) {
      if (((k & found) == prefix) & (k != kStays) & (k != kGoes)) atomicAdd(&hist[(k >> shift) & digit], 1);
    };
    if constexpr (PER > 0) {
#pragma unroll
      for (int j = 0; j < PER; ++j) count(key[j]);
    } else {
      for (int64_t q = tid; q < fours; q += THREADS) {
        uint32_t k[4];
        keys_of(q, k);
#pragma unroll
        for (int i = 0; i < 4; ++i) count(k[i]);
      }
    }
    __syncthreads();
    // the digit of the rest-th one
    int own[kOwn], sum[1] = {0};
#pragma unroll
    for (int i = 0; i < kOwn; ++i) sum[0] += own[i] = hist[tid * kOwn + i];
    int before = Scan<THREADS, 1>(sum, red).before[0];
    if (before < rest && rest <= before + sum[0]) {
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        if (before < rest && rest <= before + own[i]) {
          chosen[0] = tid * kOwn + i;
          chosen[1] = rest - before;
          chosen[2] = own[i];
        }
        before += own[i];
      }
    }
    __syncthreads();
    prefix |= (uint32_t)chosen[0] << shift;
    found |= digit << shift;
    rest = chosen[1];
    if (shift == 0 || chosen[2] == rest) break;
    bits = shift == kFirstShift ? 11 : 10;
    shift -= bits;
  }

  // In order, kRun slots a thread: 00 goes, 01 equal to the prefix, 10 stays, 11 no slot.
  auto code_of = [&](const uint32_t* k, int64_t four) {
    uint32_t code = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t m = k[i] & found;
      const uint32_t c = m < prefix ? 0u : m == prefix ? 1u : 2u;
      code |= (4 * four + i < len ? c : 3u) << (2 * i);
    }
    return (uint8_t)code;
  };
  int32_t* holes = few ? few_to : to + unit * max_pairs;
  int32_t* movers = few ? few_from : from + unit * max_pairs;
  int done[4] = {0, 0, 0, 0};  // of the slots before this round's
  // The round of the slots from `base` on, their codes in place.
  auto round = [&](int64_t base) {
    __syncthreads();
    const uint64_t w = reinterpret_cast<const Codes*>(codes)[tid];
    constexpr uint64_t kPairs = kRun == 32 ? 0x5555555555555555ull : kRun == 16 ? 0x55555555ull : 0x55ull;
    const uint64_t b0 = w & kPairs, b1 = (w >> 1) & kPairs;
    const uint64_t lower = ~(b0 | b1) & kPairs, equal = b0 & ~b1, higher = b1 & ~b0;
    const int64_t t0 = base + (int64_t)tid * kRun;
    const int below = (int)max((int64_t)0, min((int64_t)kRun, keep - t0));  // of these slots, below the budget
    const uint64_t front = below == 32 ? ~0ull : (1ull << (2 * below)) - 1;
    // dropped ones below the budget, kept ones past it, and the equal ones on either side
    const int n[4] = {(int)__popcll(lower & front), (int)__popcll(higher & ~front), (int)__popcll(equal & front),
                      (int)__popcll(equal & ~front)};
    const Scan<THREADS, 4> scan(n, red);
    // of the equal ones the first `rest` go
    const int seen = done[2] + done[3] + scan.before[2] + scan.before[3];
    uint64_t goes = lower, left = equal;
    for (int i = min(max(rest - seen, 0), n[2] + n[3]); i > 0; --i) {
      goes |= left & (0 - left);
      left &= left - 1;
    }
    const int front_total = done[2] + scan.total[2];  // whole only once past the budget, where it is used
    int hole = done[0] + scan.before[0] + min(done[2] + scan.before[2], rest);
    int mover = done[1] + scan.before[1] + done[3] + scan.before[3] - max(0, min(seen, rest) - min(front_total, rest));
    for (uint64_t h = goes & front; h != 0; h &= h - 1) holes[hole++] = (int32_t)(t0 + (__ffsll((long long)h) - 1) / 2);
    for (uint64_t m = (higher | left) & ~front; m != 0; m &= m - 1)
      movers[mover++] = (int32_t)(t0 + (__ffsll((long long)m) - 1) / 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) done[i] += scan.total[i];
  };
  if constexpr (PER > 0) {
#pragma unroll
    for (int j = 0; j < kFours; j += kRun / 4) {
      if (j > 0) __syncthreads();
#pragma unroll
      for (int r = 0; r < kRun / 4; ++r)
        codes[r * THREADS + tid] = code_of(&key[4 * (j + r)], (int64_t)(j + r) * THREADS + tid);
      round((int64_t)4 * j * THREADS);
    }
  } else {
    for (int64_t base = 0; base < len; base += (int64_t)THREADS * kRun) {
      __syncthreads();
      for (int r = 0; r < kRun / 4; ++r) {
        const int64_t q = base / 4 + r * THREADS + tid;
        uint32_t k[4] = {kStays, kStays, kStays, kStays};
        if (q < fours) keys_of(q, k);
        codes[r * THREADS + tid] = code_of(k, q);
      }
      round(base);
    }
  }
  const int count = done[0] + min(done[2], rest);
  if (tid == 0) counts[unit] = count;
  if (!few) return;
  __syncthreads();
  move_rows<THREADS, 1>(a.pages, table, head, few_to, few_from, 0, count, few_rows);
}

constexpr int kMoveThreads = 256;
constexpr int kMoveAhead = 4;

__global__ __launch_bounds__(kMoveThreads) void kv_move_kernel(const KvEvict a, const int32_t* to, const int32_t* from,
                                                               const int32_t* counts, int64_t max_pairs) {
  __shared__ int64_t rows[kPairs][2];
  const int64_t units = a.seqs * a.pages.heads;
  for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const int64_t s = unit / a.pages.heads, n = counts[unit];
    // runs of kPairs pairs, one workgroup each in turn
    for (int64_t p = (int64_t)blockIdx.y * kPairs; p < n; p += (int64_t)gridDim.y * kPairs)
      move_rows<kMoveThreads, kMoveAhead>(a.pages, a.tables + s * a.table_stride, (int)(unit - s * a.pages.heads),
                                          to + unit * max_pairs, from + unit * max_pairs, p, min(p + kPairs, n), rows);
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
  return (units * ((size_t)max_pairs(a) * 2 + 1) * 4 + 15) / 16 * 16;
}

hipError_t launch_kv_evict(const KvEvict& a, void* workspace, hipStream_t stream) {
  if (a.seqs == 0) return hipSuccess;
  const int64_t units = a.seqs * a.pages.heads, pairs = max_pairs(a);
  int32_t* to = static_cast<int32_t*>(workspace);
  int32_t* from = to + units * pairs;
  int32_t* counts = from + units * pairs;
  const int few = pairs <= kFewPairs;
  const dim3 grid((unsigned)a.seqs, (unsigned)a.pages.heads);
  // The fewest slots a thread that hold what the tables can name: a variant goes through all of its
  // slots whatever the lengths are (64 sequences of 2,064 slots, 16 pairs, us a call: 16 slots a thread
  // 15.8, 32 26.2, 64 58.8; of 1,024: 4 slots 11.0, 16 15.0).  Without registers places and weights
  // are read again in every pass (9,000 slots: 32 a thread 28.8, none 48; 8 sequences of 16,384: 22.2 and
  // 31.2; of 32,768: 64 a thread 37.2, none 49.4), which is slower at these limits, though not for
  // sequences far shorter than their tables (2,064 slots: none 29.8).
  if (a.max_length <= 1024)
    kv_select_kernel<256, 4><<<grid, 256, 0, stream>>>(a, to, from, counts, pairs, few);
  else if (a.max_length <= 4096)
    kv_select_kernel<256, 16><<<grid, 256, 0, stream>>>(a, to, from, counts, pairs, few);
  else if (a.max_length <= 16384)
    kv_select_kernel<512, 32><<<grid, 512, 0, stream>>>(a, to, from, counts, pairs, few);
  else if (a.max_length <= 32768)
    kv_select_kernel<512, 64><<<grid, 512, 0, stream>>>(a, to, from, counts, pairs, few);
  else
    kv_select_kernel<1024, 0><<<grid, 1024, 0, stream>>>(a, to, from, counts, pairs, few);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || few) return e;
  // a workgroup per run of pairs, up to some rounds of the whole machine's
  const int64_t most = std::max<int64_t>(1, 16384 / units);
  const int64_t y = std::min(most, (pairs + kPairs - 1) / kPairs);
  const int64_t x = std::min<int64_t>(units, 0xffffffffu / kMoveThreads);  // fewer than 2^32 threads
  kv_move_kernel<<<dim3((unsigned)x, (unsigned)y), kMoveThreads, 0, stream>>>(a, to, from, counts, pairs);
  return hipGetLastError();
}

}  // namespace nve_amd
