// sample_select.cuh -- sampling a row of logits from nothing but the row: cuts found by shrinking the
// range that they are in, whatever its values are (sample.hip says what comes here).
#pragma once

#include <math.h>

#include "kv_common.cuh"
#include "sample_launch.hpp"

namespace nve_amd {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;

// What is kept of a row: values above `at`, and the first `ties` of those equal to it.
struct Cut {
  float at;
  int64_t ties;
};

struct SelectShared {
  uint32_t count[kBins];
  unsigned long long mass[kBins];
  double sum[kWaves];
  int64_t whole[kWaves];
  float low[kWaves], high[kWaves];
  // of the bin that was looked for
  int bin;
  int64_t before_count;
  unsigned long long before_mass;
};

template <int DT>
struct Row {
  const kv_elem<DT>* p;
  int64_t n;
  double inverse;  // 1 / T
  float top;
  double mass_scale;

  // No number counts as minus infinity.
  __device__ __forceinline__ float value(int64_t i) const {
    const float x = (float)p[i];
    return x == x ? x : -INFINITY;
  }
  __device__ __forceinline__ double weight(float x) const {
    if (x == top) return 1.0;
    if (top == INFINITY || x == -INFINITY) return 0.0;
    return exp(((double)x - (double)top) * inverse);
  }
  // A weight, 1 at most, times 2^shift, 2^51 at most, rounded by adding 2^52; those of a row sum to less than 2^62.
  __device__ __forceinline__ unsigned long long mass(float x) const {
    const double w = weight(x) * mass_scale + 0x1p52;
    return (unsigned long long)__double_as_longlong(w) & ((1ull << 52) - 1);
  }
};

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) x += __shfl_xor(x, m);
  return x;
}

// A value between the finite ones and infinity stands for infinity.
__device__ __forceinline__ double finite(float x) { return x == INFINITY ? 0x1p129 : (double)x; }

// Values from `high` down to `low` in kBins bins of one width; bin 0 has `high`, the last one `low`.
struct Bins {
  double high, scale;
  __device__ __forceinline__ Bins(float low, float high_)
      : high(finite(high_)), scale((kBins - 0.001) / (finite(high_) - finite(low))) {}
  __device__ __forceinline__ int of(float x) const { return min(kBins - 1, (int)((high - finite(x)) * scale)); }
};

// Least and greatest value of the row within [low, high] that `f` says yes to; all threads get them.
template <int DT, typename F>
__device__ __forceinline__ void range_of(const Row<DT>& r, SelectShared& s, float& low, float& high, F f) {
  float lo = INFINITY, hi = -INFINITY;
  for (int64_t i = threadIdx.x; i < r.n; i += kThreads) {
    const float x = r.value(i);
    if (f(x)) {
      lo = fminf(lo, x);
      hi = fmaxf(hi, x);
    }
  }
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) {
    lo = fminf(lo, __shfl_xor(lo, m));
    hi = fmaxf(hi, __shfl_xor(hi, m));
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    s.low[threadIdx.x >> 6] = lo;
    s.high[threadIdx.x >> 6] = hi;
  }
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) {
    lo = fminf(lo, s.low[w]);
    hi = fmaxf(hi, s.high[w]);
  }
  low = lo;
  high = hi;
}

// The first place in the order at which the count (BY_MASS: the mass) of what is before and at it
// reaches `target`, among the values in [low, high]; false: it never does.  mass: what is above the cut.
template <int DT, bool BY_MASS>
__device__ __forceinline__ bool select(const Row<DT>& r, SelectShared& s, float low, float high, unsigned long long target,
                                       Cut& cut, unsigned long long& above_mass) {
  const int tid = threadIdx.x;
  unsigned long long above_count = 0;
  above_mass = 0;
  while (low < high) {
    const Bins bins(low, high);
    for (int b = tid; b < kBins; b += kThreads) {
      s.count[b] = 0;
      s.mass[b] = 0;
    }
    if (tid == 0) s.bin = -1;
    __syncthreads();
    for (int64_t i = tid; i < r.n; i += kThreads) {
      const float x = r.value(i);
      if (x >= low && x <= high) {
        const int b = bins.of(x);
        atomicAdd(&s.count[b], 1u);
        atomicAdd(&s.mass[b], r.mass(x));
      }
    }
    __syncthreads();
    // one wave goes through the bins, 64 at a time
    if (tid < 64) {
      unsigned long long c = above_count, m = above_mass;
      for (int b0 = 0; b0 < kBins; b0 += 64) {
        const unsigned long long own_c = s.count[b0 + tid], own_m = s.mass[b0 + tid];
        unsigned long long sc = own_c, sm = own_m;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const unsigned long long oc = __shfl_up(sc, d), om = __shfl_up(sm, d);
          if (tid >= d) {
            sc += oc;
            sm += om;
          }
        }
        const bool here = (BY_MASS ? m + sm : c + sc) >= target && own_c > 0;
        const uint64_t any = __ballot(here);
        if (any) {
          if (tid == __builtin_ctzll(any)) {
            s.bin = b0 + tid;
            s.before_count = (int64_t)(c + sc - own_c);
            s.before_mass = m + sm - own_m;
          }
          break;
        }
        c += __shfl(sc, 63);
        m += __shfl(sm, 63);
      }
    }
    __syncthreads();
    const int bin = s.bin;
    if (bin < 0) return false;
    above_count = (unsigned long long)s.before_count;
    above_mass = s.before_mass;
    const float l = low, h = high;
    range_of(r, s, low, high, [&](float x) { return x >= l && x <= h && bins.of(x) == bin; });
  }
  cut.at = low;
  if constexpr (BY_MASS) {
    const unsigned long long each = r.mass(low);
    const unsigned long long left = target > above_mass ? target - above_mass : 1;
    if (each == 0) return false;
    cut.ties = (int64_t)((left + each - 1) / each);
  } else {
    cut.ties = (int64_t)(target - above_count);
  }
  return true;
}

// A row from nothing but its logits.
template <int DT>
__device__ __forceinline__ void sample_row(const Sample& a, const int shift, const int64_t row, SelectShared& s) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float t = a.temperature ? a.temperature[row] : a.temperature_all;
  const int64_t k = a.top_k ? a.top_k[row] : a.top_k_all;
  const float p = a.top_p ? a.top_p[row] : a.top_p_all;
  const float min_p = a.min_p ? a.min_p[row] : a.min_p_all;
  Row<DT> r;
  r.p = reinterpret_cast<const kv_elem<DT>*>(a.logits) + row * a.row_stride;
  r.n = a.vocab;
  r.mass_scale = ldexp(1.0, shift);
  float least;
  range_of(r, s, least, r.top, [](float x) { return x > -INFINITY; });
  if (!(r.top > -INFINITY)) {
    if (tid == 0) a.tokens[row] = -1;
    return;
  }
  const bool greedy = !(t > 0.0f);
  r.inverse = greedy ? 0.0 : 1.0 / (double)t;

  Cut cut{-INFINITY, r.n};
  if (greedy) {
    cut = {r.top, 1};
  } else {
    unsigned long long above = 0;
    if (k > 0 && k < r.n) select<DT, false>(r, s, least, r.top, (unsigned long long)k, cut, above);
    if (p < 1.0f) {
      unsigned long long total;
      if (cut.at > -INFINITY) {
        total = above + (unsigned long long)cut.ties * r.mass(cut.at);
      } else {
        unsigned long long sum = 0;
        for (int64_t i = tid; i < r.n; i += kThreads) sum += r.mass(r.value(i));
#pragma unroll
        for (int m = 32; m > 0; m >>= 1) sum += __shfl_xor(sum, m);
        __syncthreads();
        if (lane == 0) s.whole[wave] = (int64_t)sum;
        __syncthreads();
        total = 0;
        for (int w = 0; w < kWaves; ++w) total += (unsigned long long)s.whole[w];
      }
      const double target = fmax(ceil((double)p * (double)total), 1.0);
      Cut nucleus;
      const float low = cut.at > -INFINITY ? cut.at : least;
      if (select<DT, true>(r, s, low, r.top, (unsigned long long)target, nucleus, above)) {
        if (nucleus.at > cut.at) cut = nucleus;
        else cut.ties = min(cut.ties, nucleus.ties);
      }
    }
  }
  const double limit = min_p > 0.0f ? fmin((double)min_p, 1.0) : 0.0;
  const double tie = r.weight(cut.at) >= limit ? r.weight(cut.at) : 0.0;

  // narrows [first, last) down to a wave's 64 values, by the sums of 16 runs of it
  int64_t first = 0, last = r.n, ties_before = 0;
  double before = 0.0, target = -1.0;
  const double u = a.u[row] > 0.0f ? (double)a.u[row] : 0.0;
  for (;;) {
    const int64_t run = ((last - first + kWaves - 1) / kWaves + 63) / 64 * 64;
    const int64_t b = first + wave * run, e = min(b + run, last);
    double sum = 0.0;
    int64_t equal = 0;
    for (int64_t i = b + lane; i < e; i += 64) {
      const float x = r.value(i);
      if (x > cut.at) {
        const double w = r.weight(x);
        sum += w >= limit ? w : 0.0;
      }
      equal += x == cut.at;
    }
    sum = wave_sum(sum);
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) equal += __shfl_xor(equal, m);
    __syncthreads();
    if (lane == 0) {
      s.sum[wave] = sum;
      s.whole[wave] = equal;
    }
    __syncthreads();
    // every thread goes through the 16 sums
    double at = before, end = before;
    int64_t ties = ties_before;
    if (target < 0.0) {
      for (int w = 0; w < kWaves; ++w) {
        const int64_t kept = max((int64_t)0, min(s.whole[w], cut.ties - ties));
        end += s.sum[w] + (double)kept * tie;
        ties += s.whole[w];
      }
      target = u * end;
      ties = ties_before;
    }
    int found = -1;
    double found_before = 0.0;
    int64_t found_ties = 0;
    for (int w = 0; w < kWaves; ++w) {
      const int64_t kept = max((int64_t)0, min(s.whole[w], cut.ties - ties));
      const double mass = s.sum[w] + (double)kept * tie;
      if (mass > 0.0) {  // the last one with any, where none reaches the target
        found = w;
        found_before = at;
        found_ties = ties;
        if (at + mass > target) break;
      }
      at += mass;
      ties += s.whole[w];
    }
    if (run == 64) {  // a value a lane
      if (wave == found) {
        const float x = b + lane < e ? r.value(b + lane) : -INFINITY;
        const bool same = x == cut.at && b + lane < e;
        const uint64_t equals = __ballot(same);
        const int64_t rank = found_ties + __popcll(equals & ((1ull << lane) - 1));
        const double w0 = r.weight(x);
        double w = same ? (rank < cut.ties ? tie : 0.0) : x > cut.at && w0 >= limit ? w0 : 0.0;
        double scan = w;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const double o = __shfl_up(scan, d);
          if (lane >= d) scan += o;
        }
        const uint64_t over = __ballot(w > 0.0 && found_before + scan > target), any = __ballot(w > 0.0);
        if (lane == 0) a.tokens[row] = b + (over ? __builtin_ctzll(over) : 63 - __builtin_clzll(any));
      }
      return;
    }
    first = first + found * run;
    last = min(first + run, last);
    before = found_before;
    ties_before = found_ties;
  }
}

}  // namespace nve_amd
