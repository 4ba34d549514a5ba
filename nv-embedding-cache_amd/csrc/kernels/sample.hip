// sample.hip -- a token for every row of logits from one random number, after temperature, top-k,
// top-p and min-p.
//
// With w_i = exp((x_i - max) / T) the tokens that are kept are the first ones in the order (value
// descending, index ascending): top-k's of them, top-p's (those whose preceding sum is below p times
// the sum of top-k's) and min-p's (w_i >= min_p, as the largest w is 1).  The token is the first index
// at which the kept weights' running sum, in the vocabulary's order, exceeds u times their total.
//
// Weights are 64-bit: a token's probability may be 1e-6, and a sum in 32 bits would give some
// tokens' share of the random numbers to their neighbours.  A vector instruction in 64 bits takes as
// long here as one in 32.  Sums that pick a cut are integers (weights times 2^shift), so that the order
// of the LDS additions changes nothing.
//
// Bound: the logits' bytes, read once.  scan_kernel reads them and leaves the maximum of every 64
// neighbours (a group) and, for rows that need the whole distribution's mass, the mass of every wave's
// unit.  pick_kernel, a workgroup a row, goes on with these:
//   nothing is cut off     the unit that u times the mass falls into is read again
//   few tokens are kept    k maxima above a value are k tokens above it, and weights of maxima that sum
//                          to p of all are a nucleus: only groups whose maximum is above such a value
//                          are read again, and their values above it sorted
//   a wide nucleus         a histogram of the row's masses, then the masses of units above the cut's bin
// select() serves what is left (a large top-k, infinities, many equals at a wide cut, vocabularies of
// more than 2^19): it shrinks the range that the cut is in by histograms, from nothing but the row.
#include <math.h>

#include <algorithm>

#include "../dtypes.hpp"
#include "kv_common.cuh"
#include "sample_launch.hpp"
#include "sample_select.cuh"

namespace nve_amd {

namespace {

using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;

constexpr int kCandidates = 2048;        // sorted at most
constexpr int kMostGroups = 8192;
constexpr int kMostUnits = 512;
constexpr int kPieces = 4;               // 16-byte pieces of a lane in a unit
constexpr int64_t kMostVocab = 1 << 19;  // of the two kernels: 8192 groups, 512 units

// What scan_kernel leaves of the rows of a launch.
struct Left {
  int64_t groups, units;
  int32_t group;      // values
  float* group_top;   // [rows, groups]
  float* unit_top;    // [rows, units]
  double* unit_mass;  // [rows, units], relative to the unit's maximum
};

// A row's limits.
struct Limits {
  bool greedy, k_on, p_on, low_on;
  int64_t k;
  double p, low, scale;  // scale: log2(e) / T
  __device__ __forceinline__ Limits(const Sample& a, int64_t row) {
    const float t = a.temperature ? a.temperature[row] : a.temperature_all;
    const float pf = a.top_p ? a.top_p[row] : a.top_p_all;
    const float lf = a.min_p ? a.min_p[row] : a.min_p_all;
    k = a.top_k ? a.top_k[row] : a.top_k_all;
    greedy = !(t > 0.0f);
    k_on = k > 0 && k < a.vocab;
    p_on = pf < 1.0f;
    low_on = lf > 0.0f;
    p = pf;
    low = low_on ? fmin((double)lf, 1.0) : 0.0;
    scale = greedy ? 0.0 : 1.4426950408889634 / (double)t;
  }
  __device__ __forceinline__ bool all_mass() const { return !greedy && !k_on && (p_on || !low_on); }
};

// 2^z for z <= 0, to some 2^-52: a table of 2^(j / 32) and the exponential's series up to the fifth power for
// the rest, |r| <= 1/64, whose next term is (ln 2 / 64)^6 / 720 = 2.2e-15.  2^-1100 and less is 0, and so
// is what is no number.
struct Exp2 {
  const double* table;
  static __device__ __forceinline__ void fill(double* t) {
    if (threadIdx.x < 32) t[threadIdx.x] = exp2(threadIdx.x / 32.0);
  }
  __device__ __forceinline__ double operator()(double z) const {
    z = fmax(z, -1100.0);
    const double t = z + 0x1.8p47;  // a multiple of 1/32
    const int n = (int)__double_as_longlong(t);
    const double r = z - (t - 0x1.8p47);
    double y = fma(r, 0.0013333558146428443, 0.009618129107628477);
    y = fma(r, y, 0.05550410866482158);
    y = fma(r, y, 0.2402265069591007);
    y = fma(r, y, 0.6931471805599453);
    y = fma(r, y, 1.0);
    return ldexp(table[n & 31] * y, n >> 5);
  }
};

// A lane's 16 bytes of a row from `first` on; what is past the row's end, or no number, is minus infinity
// (or stays a NaN, which every comparison leaves out).
template <int DT>
struct Piece {
  static constexpr int kValues = 16 / value_elem_bytes(DT);
  kv_elem<DT> v[kValues];
  __device__ __forceinline__ void load(const kv_elem<DT>* row, int64_t first, int64_t n) {
    typedef u32x4 __attribute__((aligned(2))) any;  // a row may start at any element
    if (first + kValues <= n) {
      const u32x4 w = *reinterpret_cast<const any*>(row + first);
      __builtin_memcpy(v, &w, 16);
    } else {
#pragma unroll
      for (int i = 0; i < kValues; ++i) v[i] = first + i < n ? row[first + i] : (kv_elem<DT>)-INFINITY;
    }
  }
  __device__ __forceinline__ float operator[](int i) const { return (float)v[i]; }
};

template <int DT>
constexpr int unit_values() {
  return kPieces * 64 * Piece<DT>::kValues;
}

// Maxima over 2, 4, 8, 16 or 64 neighbouring lanes.
template <int CTRL>
__device__ __forceinline__ float max_with(float x) {
  return fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(x), __float_as_int(x), CTRL, 0xf, 0xf, false)));
}
template <int LANES>
__device__ __forceinline__ float lanes_max(float x) {
  x = max_with<0xb1>(x);                               // the neighbour
  if constexpr (LANES >= 4) x = max_with<0x4e>(x);     // the pair beside
  if constexpr (LANES >= 8) x = max_with<0x141>(x);    // the four beside: half a row mirrored
  if constexpr (LANES >= 16) x = max_with<0x140>(x);   // a row mirrored
  if constexpr (LANES == 64) {
    x = fmaxf(x, __shfl_xor(x, 16));
    x = fmaxf(x, __shfl_xor(x, 32));
  }
  return x;
}

// ---------------------------------------------------------------------------
// the first kernel: a unit a wave
// ---------------------------------------------------------------------------
constexpr int kScanThreads = 256;

template <int DT, int GROUP>
__global__ __launch_bounds__(kScanThreads) void scan_kernel(const Sample a, const Left l, const int blocks) {
  constexpr int kValues = Piece<DT>::kValues, kLanes = GROUP / kValues;
  __shared__ double table[32];
  const int lane = threadIdx.x & 63;
  const int64_t row = blockIdx.x / blocks;
  const int64_t unit = (int64_t)(blockIdx.x - row * blocks) * (kScanThreads / 64) + (threadIdx.x >> 6);
  const Limits limits(a, row);
  if (limits.all_mass()) Exp2::fill(table);
  __syncthreads();
  if (unit >= l.units) return;
  const kv_elem<DT>* p = reinterpret_cast<const kv_elem<DT>*>(a.logits) + row * a.row_stride;
  const int64_t base = unit * unit_values<DT>() + lane * kValues;
  Piece<DT> x[kPieces];
#pragma unroll
  for (int j = 0; j < kPieces; ++j) x[j].load(p, base + j * 64 * kValues, a.vocab);
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    float m = x[j][0];
#pragma unroll
    for (int i = 1; i < kValues; ++i) m = fmaxf(m, x[j][i]);
    m = lanes_max<kLanes>(fmaxf(m, -INFINITY));
    const int64_t group = (base + j * 64 * kValues) / GROUP;
    if (lane % kLanes == 0 && group < l.groups) l.group_top[row * l.groups + group] = m;
    top = fmaxf(top, m);
  }
  if (!limits.all_mass()) return;
  top = lanes_max<64>(top);
  const Exp2 exp2_of{table};
  const double high = top;
  double sum = 0.0;
  if (top > -INFINITY && top < INFINITY) {
#pragma unroll
    for (int j = 0; j < kPieces; ++j)
#pragma unroll
      for (int i = 0; i < kValues; ++i) sum += exp2_of(((double)x[j][i] - high) * limits.scale);
    sum = wave_sum(sum);
  }
  if (lane == 0) {
    l.unit_top[row * l.units + unit] = top;
    l.unit_mass[row * l.units + unit] = sum;
  }
}

// ---------------------------------------------------------------------------
// the second kernel: a row a workgroup
// ---------------------------------------------------------------------------
struct PickShared {
  uint64_t keys[kCandidates];    // in the vocabulary's order
  uint64_t sorted[kCandidates];  // the greatest first
  union {
    uint16_t groups[kMostGroups];
    struct {
      uint32_t count[kBins];
      unsigned long long mass[kBins];
    };
  };
  double unit[kMostUnits];
  double red_sum[kWaves];
  unsigned long long red_mass[kWaves];
  int red_count[kWaves];
  float red_low[kWaves], red_high[kWaves];
  double table[32];
  int found, last, bin, bin2;
  int n;
  double before;
  unsigned long long before_mass;
  uint64_t cut;
};

union AnyShared {
  SelectShared select;
  PickShared pick;
};

// The order of tokens as one number: the value, then the lower index first.  Both zeros are one value.
__device__ __forceinline__ uint64_t key_of(float x, int64_t index) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  const uint32_t o = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  return (uint64_t)o << 32 | (uint32_t)~(uint32_t)index;
}
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ int64_t index_of(uint64_t key) { return (uint32_t)~(uint32_t)key; }

// x of the threads up to and including this one, added in one order; total: of all.
template <typename T>
__device__ __forceinline__ T block_scan(T x, T* red, T& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const T o = __shfl_up(x, d);
    if (lane >= d) x += o;
  }
  __syncthreads();
  if (lane == 63) red[wave] = x;
  __syncthreads();
  T before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const T r = red[w];
    if (w < wave) before += r;
    total += r;
  }
  return before + x;
}

// The first of n <= 2 kThreads items at which the running sum of their weights, from `base` on, exceeds the
// target; the last one with a weight where none does.  share: the target is u times the sum.
template <typename F>
__device__ __forceinline__ int pick_item(PickShared& s, int n, double base, double target, bool share, F weight) {
  const int i = 2 * threadIdx.x;
  const double w0 = i < n ? weight(i) : 0.0, w1 = i + 1 < n ? weight(i + 1) : 0.0;
  double total;
  const double end = block_scan(w0 + w1, s.red_sum, total);
  if (threadIdx.x == 0) {
    s.found = 1 << 30;
    s.last = 0;
  }
  __syncthreads();
  if (share) target *= total;
  if (w0 > 0.0 && base + (end - w1) > target) atomicMin(&s.found, i);
  else if (w1 > 0.0 && base + end > target) atomicMin(&s.found, i + 1);
  if (w1 > 0.0) atomicMax(&s.last, i + 1);
  else if (w0 > 0.0) atomicMax(&s.last, i);
  __syncthreads();
  return s.found < (1 << 30) ? s.found : s.last;
}

// Sorts n <= kCandidates keys, the greatest first; those behind them up to a power of two become 0.
__device__ __forceinline__ void sort_keys(uint64_t* keys, int n) {
  const int tid = threadIdx.x;
  int size2 = 2;
  while (size2 < n) size2 <<= 1;
  for (int i = n + tid; i < size2; i += kThreads) keys[i] = 0;
  __syncthreads();
  for (int size = 2; size <= size2; size <<= 1) {
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      if (tid < size2 / 2) {
        const int low = 2 * tid - (tid & (stride - 1)), high = low + stride;
        const uint64_t x = keys[low], y = keys[high];
        if ((x < y) == ((low & size) == 0)) {
          keys[low] = y;
          keys[high] = x;
        }
      }
      __syncthreads();
    }
  }
}
static_assert(kCandidates == 2 * kThreads);

// kBins bins of one width from `high` down; the last one has all that is below, and what is no number.
struct Steps {
  float high, scale;
  __device__ __forceinline__ Steps(float high, float low) : high(high) {
    const float width = high - low;
    scale = width > 0.0f ? fminf((kBins - 0.1f) / width, 3e38f) : 3e38f;
  }
  __device__ __forceinline__ int of(float x) const { return (int)fminf((high - x) * scale, kBins - 1.0f); }
};

template <int DT, int GROUP>
struct Pick {
  static constexpr int kValues = Piece<DT>::kValues, kLanes = GROUP / kValues, kUnit = unit_values<DT>();
  const Sample& a;
  const Left& l;
  const Limits& limits;
  PickShared& s;
  const int64_t row;
  const kv_elem<DT>* p;
  float top;
  double high, mass_scale;
  double u;

  __device__ __forceinline__ double weight(float x) const {
    return Exp2{s.table}(((double)x - high) * limits.scale);
  }
  __device__ __forceinline__ unsigned long long mass_of(double w) const {
    return (unsigned long long)__double_as_longlong(w * mass_scale + 0x1p52) & ((1ull << 52) - 1);
  }
  __device__ __forceinline__ void answer(int64_t token) const {
    if (threadIdx.x == 0) a.tokens[row] = token;
  }

  // The bin at which the running sum of the bins' numbers reaches the target, or -1; its predecessors' sum.
  template <typename T>
  __device__ __forceinline__ int bin_at(const T* bins, T target, T& before) const {
    const int tid = threadIdx.x;
    const unsigned long long x0 = bins[2 * tid], x1 = bins[2 * tid + 1];
    unsigned long long total;
    const unsigned long long end = block_scan<unsigned long long>(x0 + x1, s.red_mass, total);
    if (tid == 0) s.bin = -1;
    __syncthreads();
    const unsigned long long b1 = end - x1, b0 = b1 - x0, t = target;
    if (b0 < t && b1 >= t) {
      s.bin = 2 * tid;
      s.before_mass = b0;
    } else if (b1 < t && end >= t) {
      s.bin = 2 * tid + 1;
      s.before_mass = b1;
    }
    __syncthreads();
    before = (T)s.before_mass;
    return s.bin;
  }

  // The token within a unit: values from `cut` on, the least weight `low`.
  __device__ __forceinline__ int64_t pick_in_unit(int64_t unit, double base, double target, uint64_t cut, double low) const {
    const int64_t first = unit * kUnit;
    const int n = (int)min((int64_t)kUnit, a.vocab - first);
    return first + pick_item(s, n, base, target, false, [&](int i) {
      const float x = (float)p[first + i];
      if (!(x > -INFINITY) || key_of(x, first + i) < cut) return 0.0;
      const double w = weight(x);
      return w >= low ? w : 0.0;
    });
  }

  // The unit whose mass the share u falls into (s.unit has the units' masses), and the token in it.
  __device__ __forceinline__ void pick_unit(uint64_t cut, double low) const {
    const int tid = threadIdx.x, n = (int)l.units;
    const int unit = pick_item(s, n, 0.0, u, true, [&](int i) { return s.unit[i]; });
    // the sum before it, and the target, from the same numbers
    double total;
    const double own = tid < n ? s.unit[tid] : 0.0;
    const double end = block_scan(own, s.red_sum, total);
    __syncthreads();
    if (tid == unit) s.before = end - own;
    __syncthreads();
    answer(pick_in_unit(unit, s.before, u * total, cut, low));
  }

  // A wide nucleus (target: the mass it needs, in units of 2^-shift), or the tokens of weight `low` and more
  // (target 0).  all: the mass of all.  false: not decided here.
  __device__ __forceinline__ bool wide(unsigned long long target, double all) const {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // a nucleus leaves out (1 - p) of the mass at most, so its least weight is at least that over the vocabulary
    float least = -INFINITY;
    if (target > 0) {
      const double depth = log2((double)a.vocab / ((1.0 - limits.p) * all)) / limits.scale;
      if (!(depth < 1e30)) return false;
      least = (float)(high - fmax(depth, 0.0) * 1.0001 - 1e-6 * fabs(high));
      if (!(least > -3e38f)) return false;
    }
    const Steps steps(top, target > 0 ? least : top);
    int bin = kBins;  // what is before it is kept whole
    unsigned long long above = 0;
    if (target > 0) {
      for (int i = tid; i < kBins; i += kThreads) s.mass[i] = 0;
      __syncthreads();
      for (int64_t unit = wave; unit < l.units; unit += kWaves) {
        const int64_t base = unit * kUnit + lane * kValues;
        Piece<DT> x[kPieces];
#pragma unroll
        for (int j = 0; j < kPieces; ++j) x[j].load(p, base + j * 64 * kValues, a.vocab);
#pragma unroll
        for (int j = 0; j < kPieces; ++j)
#pragma unroll
          for (int i = 0; i < kValues; ++i)
            if (x[j][i] >= least) atomicAdd(&s.mass[steps.of(x[j][i])], mass_of(weight(x[j][i])));
      }
      __syncthreads();
      bin = bin_at<unsigned long long>(s.mass, target, above);
      if (bin < 0) return false;
    }
    if (tid == 0) s.n = 0;
    __syncthreads();
    for (int64_t unit = wave; unit < l.units; unit += kWaves) {
      const int64_t base = unit * kUnit + lane * kValues;
      Piece<DT> x[kPieces];
#pragma unroll
      for (int j = 0; j < kPieces; ++j) x[j].load(p, base + j * 64 * kValues, a.vocab);
      double sum = 0.0;
#pragma unroll
      for (int j = 0; j < kPieces; ++j)
#pragma unroll
        for (int i = 0; i < kValues; ++i) {
          const float v = x[j][i];
          const int b = target > 0 ? steps.of(v) : 0;
          if (b == bin && v >= least) {
            const int at = atomicAdd(&s.n, 1);
            if (at < kCandidates) s.sorted[at] = key_of(v, base + j * 64 * kValues + i);
          } else if (b < bin && v > -INFINITY) {
            const double w = weight(v);
            sum += w >= limits.low ? w : 0.0;
          }
        }
      sum = wave_sum(sum);
      if (lane == 0) s.unit[unit] = sum;
    }
    __syncthreads();
    uint64_t cut = 0;
    const int n = s.n;
    if (n > kCandidates) return false;
    if (n > 0) {
      sort_keys(s.sorted, n);
      const int i = 2 * tid;
      const double w0 = i < n ? weight(value_of(s.sorted[i])) : 0.0, w1 = i + 1 < n ? weight(value_of(s.sorted[i + 1])) : 0.0;
      const unsigned long long m0 = mass_of(w0), m1 = i + 1 < n ? mass_of(w1) : 0;
      unsigned long long total;
      const unsigned long long end = above + block_scan<unsigned long long>((i < n ? m0 : 0) + m1, s.red_mass, total);
      if (tid == 0) s.cut = s.sorted[n - 1];
      __syncthreads();
      const unsigned long long b1 = end - m1, b0 = b1 - m0;
      if (i < n && b0 < target && b1 >= target) s.cut = s.sorted[i];
      else if (i + 1 < n && b1 < target && end >= target) s.cut = s.sorted[i + 1];
      __syncthreads();
      cut = s.cut;
      // the bin's kept values join their units, in the order of the sorting
      for (int unit = tid; unit < l.units; unit += kThreads) {
        double sum = s.unit[unit];
        for (int j = 0; j < n && s.sorted[j] >= cut; ++j) {
          if (index_of(s.sorted[j]) / kUnit != unit) continue;
          const double w = weight(value_of(s.sorted[j]));
          sum += w >= limits.low ? w : 0.0;
        }
        s.unit[unit] = sum;
      }
    } else if (target > 0) {
      return false;
    }
    __syncthreads();
    pick_unit(cut, limits.low);
    return true;
  }

  // false: not decided here.
  __device__ __forceinline__ bool run() {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = (int)((l.groups + kThreads - 1) / kThreads), g0 = tid * per;
    constexpr int kMostPer = kMostGroups / kThreads;
    float tops[kMostPer];
#pragma unroll
    for (int i = 0; i < kMostPer; ++i)
      tops[i] = i < per && g0 + i < l.groups ? l.group_top[row * l.groups + g0 + i] : -INFINITY;
    float lo = INFINITY, hi = -INFINITY;
#pragma unroll
    for (int i = 0; i < kMostPer; ++i) {
      hi = fmaxf(hi, tops[i]);
      if (tops[i] > -INFINITY) lo = fminf(lo, tops[i]);
    }
    hi = lanes_max<64>(hi);
    lo = -lanes_max<64>(-lo);
    if (lane == 0) {
      s.red_high[wave] = hi;
      s.red_low[wave] = lo;
    }
    Exp2::fill(s.table);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      hi = fmaxf(hi, s.red_high[w]);
      lo = fminf(lo, s.red_low[w]);
    }
    top = hi;
    high = hi;
    if (top == -INFINITY) {
      answer(-1);
      return true;
    }
    if (top == INFINITY) return false;
    u = a.u[row] > 0.0f ? (double)a.u[row] : 0.0;

    double all = 0.0;  // the mass of all, where it counts
    if (limits.all_mass()) {
      double m = 0.0;
      if (tid < l.units) {
        const float t = l.unit_top[row * l.units + tid];
        m = t > -INFINITY ? l.unit_mass[row * l.units + tid] * weight(t) : 0.0;
        s.unit[tid] = m;
      }
      block_scan(m, s.red_sum, all);
      if (!limits.p_on) {
        __syncthreads();
        pick_unit(0, 0.0);
        return true;
      }
    }

    // candidates: values in the first `limit` + 1 steps and not below `least`
    Steps steps(top, lo);
    int limit = kBins;
    float least = -INFINITY;
    unsigned long long target = 0;
    if (limits.greedy) {
      least = top;
    } else {
      if (limits.low_on && !limits.p_on && limits.scale > 0.0) {  // top-p's sums are of all of top-k's
        // a little below the least weight's value: what is between is left out by its weight
        const double low = high + log2(limits.low) / limits.scale;
        least = (float)(low - 1e-6 * fabs(low) - 1e-6 * fabs(high));
      }
      if (limits.k_on || limits.p_on) {
        for (int i = tid; i < kBins; i += kThreads) {
          s.count[i] = 0;
          s.mass[i] = 0;
        }
        __syncthreads();
        const bool by_mass = !limits.k_on;
#pragma unroll
        for (int i = 0; i < kMostPer; ++i) {
          if (tops[i] > -INFINITY) {
            const int b = steps.of(tops[i]);
            atomicAdd(&s.count[b], 1u);
            if (by_mass) atomicAdd(&s.mass[b], mass_of(weight(tops[i])));
          }
        }
        __syncthreads();
        uint32_t before;
        if (limits.k_on) {
          if (limits.k > kCandidates) return false;
          limit = bin_at<uint32_t>(s.count, (uint32_t)limits.k, before);
          if (limit < 0) return false;
        } else {
          target = (unsigned long long)fmax(ceil(limits.p * all * mass_scale), 1.0);
          unsigned long long mass_before;
          const int sure = bin_at<unsigned long long>(s.mass, target, mass_before);
          const int many = bin_at<uint32_t>(s.count, (uint32_t)min((int64_t)768, (l.groups + 1) / 2), before);
          limit = sure >= 0 && (many < 0 || sure < many) ? sure : many;
          if (limit < 0) return wide(target, all);
        }
      }
    }
    auto wanted = [&](float x) { return x >= least && x > -INFINITY && (limit >= kBins || steps.of(x) <= limit); };

    // the groups with candidates, in order
    int mine = 0;
#pragma unroll
    for (int i = 0; i < kMostPer; ++i) mine += wanted(tops[i]);
    int groups;
    int at = block_scan(mine, s.red_count, groups) - mine;
    bool few = groups <= kCandidates;
    int n = 0;
    if (few) {
#pragma unroll
      for (int i = 0; i < kMostPer; ++i)
        if (wanted(tops[i])) s.groups[at++] = (uint16_t)(g0 + i);
      __syncthreads();
      // their candidates, in order
      for (int b0 = 0; b0 < groups; b0 += kThreads / kLanes) {
        const int mine_at = b0 + tid / kLanes;
        Piece<DT> x;
        uint32_t yes = 0;
        int64_t first = 0;
        if (mine_at < groups) {
          first = (int64_t)s.groups[mine_at] * GROUP + tid % kLanes * kValues;
          x.load(p, first, a.vocab);
#pragma unroll
          for (int i = 0; i < kValues; ++i) yes |= (uint32_t)wanted(x[i]) << i;
        }
        int more;
        int to = n + block_scan((int)__popc(yes), s.red_count, more) - __popc(yes);
        if (n + more > kCandidates) {
          few = false;
          break;
        }
#pragma unroll
        for (int i = 0; i < kValues; ++i)
          if (yes >> i & 1) s.keys[to++] = key_of(x[i], first + i);
        n += more;
      }
    }
    __syncthreads();
    if (limits.greedy) {  // the first group with the maximum has the first of them
      if (few) answer(index_of(s.keys[0]));
      return few;
    }
    if (!few) {
      if (limits.k_on) return false;
      return wide(target, all);
    }

    uint64_t cut = 0;
    if (limits.k_on || limits.p_on) {
      for (int i = tid; i < n; i += kThreads) s.sorted[i] = s.keys[i];
      sort_keys(s.sorted, n);
      const int kept = limits.k_on ? (int)min((int64_t)n, limits.k) : n;
      cut = s.sorted[kept - 1];
      if (limits.p_on) {
        const int i = 2 * tid;
        const unsigned long long m0 = i < kept ? mass_of(weight(value_of(s.sorted[i]))) : 0;
        const unsigned long long m1 = i + 1 < kept ? mass_of(weight(value_of(s.sorted[i + 1]))) : 0;
        unsigned long long total;
        const unsigned long long end = block_scan<unsigned long long>(m0 + m1, s.red_mass, total);
        if (limits.k_on) target = (unsigned long long)fmax(ceil(limits.p * (double)total), 1.0);
        else if (total < target) return wide(target, all);  // the candidates are not all of the nucleus
        if (tid == 0) s.cut = cut;
        __syncthreads();
        const unsigned long long b1 = end - m1, b0 = b1 - m0;
        if (i < kept && b0 < target && b1 >= target) s.cut = s.sorted[i];
        else if (i + 1 < kept && b1 < target && end >= target) s.cut = s.sorted[i + 1];
        __syncthreads();
        cut = s.cut;
      }
    }
    const int item = pick_item(s, n, 0.0, u, true, [&](int i) {
      if (s.keys[i] < cut) return 0.0;
      const double w = weight(value_of(s.keys[i]));
      return w >= limits.low ? w : 0.0;
    });
    answer(index_of(s.keys[item]));
    return true;
  }
};

template <int DT, int GROUP>
__global__ __launch_bounds__(kThreads) void pick_kernel(const Sample a, const Left l, const int shift) {
  __shared__ AnyShared s;
  const int64_t row = blockIdx.x;
  const Limits limits(a, row);
  Pick<DT, GROUP> pick{a, l, limits, s.pick, row, reinterpret_cast<const kv_elem<DT>*>(a.logits) + row * a.row_stride};
  pick.mass_scale = ldexp(1.0, shift);
  if (pick.run()) return;
  __syncthreads();
  sample_row<DT>(a, shift, row, s.select);
}

template <int DT>
__global__ __launch_bounds__(kThreads) void select_kernel(const Sample a, const int shift) {
  __shared__ SelectShared s;
  sample_row<DT>(a, shift, blockIdx.x, s);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
// The n rows from r0 on.
Sample part(const Sample& a, int64_t r0, int64_t n) {
  Sample r = a;
  r.rows = n;
  r.logits += r0 * a.row_stride * value_elem_bytes(a.dtype);
  r.u += r0;
  r.tokens += r0;
  if (r.temperature) r.temperature += r0;
  if (r.top_k) r.top_k += r0;
  if (r.top_p) r.top_p += r0;
  if (r.min_p) r.min_p += r0;
  return r;
}

// Rows of a launch: 2^27 values, but a few hundred rows at least, whose workspace (an eighth of the values
// at most) the next launch takes over.
int64_t most_rows(const Sample& a) {
  return std::min(a.rows, std::max<int64_t>(256, ((int64_t)1 << 27) / std::max<int64_t>(a.vocab, 1024)));
}

int unit_of(int dtype) { return dtype == kF32 ? unit_values<kF32>() : unit_values<kF16>(); }

Left layout_of(const Sample& a, void* workspace, size_t* bytes) {
  Left l{};
  // small groups, so that there are many also of a small vocabulary: as many tokens as groups can be found by maxima
  l.group = a.vocab <= 65536 ? 16 : 64;
  l.groups = (a.vocab + l.group - 1) / l.group;
  l.units = (a.vocab + unit_of(a.dtype) - 1) / unit_of(a.dtype);
  uint8_t* at = static_cast<uint8_t*>(workspace);
  size_t used = 0;
  auto take = [&](size_t n) {
    void* x = at + used;
    used += (n + 15) / 16 * 16;
    return x;
  };
  const size_t rows = (size_t)most_rows(a);
  l.unit_mass = static_cast<double*>(take(rows * l.units * 8));
  l.unit_top = static_cast<float*>(take(rows * l.units * 4));
  l.group_top = static_cast<float*>(take(rows * l.groups * 4));
  *bytes = used;
  return l;
}

template <int DT>
hipError_t launch_rows(const Sample& a, const Left& l, int shift, hipStream_t stream) {
  const unsigned n = (unsigned)a.rows;
  if (a.vocab > kMostVocab) {
    select_kernel<DT><<<n, kThreads, 0, stream>>>(a, shift);
    return hipGetLastError();
  }
  const int blocks = (int)((l.units + 3) / 4);
  if (l.group == 16) {
    scan_kernel<DT, 16><<<n * blocks, kScanThreads, 0, stream>>>(a, l, blocks);
    pick_kernel<DT, 16><<<n, kThreads, 0, stream>>>(a, l, shift);
  } else {
    scan_kernel<DT, 64><<<n * blocks, kScanThreads, 0, stream>>>(a, l, blocks);
    pick_kernel<DT, 64><<<n, kThreads, 0, stream>>>(a, l, shift);
  }
  return hipGetLastError();
}

}  // namespace

size_t sample_workspace(const Sample& a) {
  size_t bytes = 0;
  if (a.rows > 0 && a.vocab <= kMostVocab) layout_of(a, nullptr, &bytes);
  return bytes;
}

hipError_t launch_sample(const Sample& a, void* workspace, hipStream_t stream) {
  if (a.rows == 0) return hipSuccess;
  size_t bytes;
  const Left l = layout_of(a, workspace, &bytes);
  // the sum of all weights is below 2^62
  int bits = 0;
  while (((int64_t)1 << bits) < a.vocab) ++bits;
  const int shift = std::min(51, 62 - bits);
  const int64_t most = most_rows(a);
  for (int64_t r0 = 0; r0 < a.rows; r0 += most) {
    const Sample b = part(a, r0, std::min(most, a.rows - r0));
    hipError_t e;
    switch (a.dtype) {
      case kF32: e = launch_rows<kF32>(b, l, shift, stream); break;
      case kF16: e = launch_rows<kF16>(b, l, shift, stream); break;
      case kBF16: e = launch_rows<kBF16>(b, l, shift, stream); break;
      default: return hipErrorInvalidValue;
    }
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace nve_amd
