// sample.hip -- a token for every row of logits from one random number, after temperature, top-k,
// top-p and min-p.
//
// With w_i = exp((x_i - max) / T) the tokens that are kept are the first ones in the order (value
// descending, index ascending): top-k's of them, top-p's (those whose preceding sum is below p times
// the sum of top-k's) and min-p's (w_i >= min_p, as the largest w is 1).  The token is the first index
// at which the kept weights' running sum, in the vocabulary's order, exceeds u times their total.
//
// Weights are 64-bit: a token's probability may be 1e-6, and a sum in 32 bits would give some
// tokens' share of the random numbers to their neighbours.  A vector instruction in 64 bits takes
// twice as long here as one in 32.  Sums that pick a cut are integers (weights times 2^shift), so that the order
// of the LDS additions changes nothing.
//
// Bound: the logits' bytes, read once.
//   scan_kernel    reads them and leaves the maximum of every 64 or 16 neighbours (a group) and, for
//                  rows that need the whole distribution's mass, the mass of every wave's unit
//   pick_kernel    a workgroup a row.  Nothing is cut off: the unit that u times the mass falls into is
//                  read again.  Few tokens are kept: k maxima above a value are k tokens above it, and
//                  maxima whose weights sum to p of all are a nucleus, so only groups with a maximum
//                  above such a value are read again, and their values above it sorted
//   slice_kernel   up to 8 workgroups (fewer where there are many rows) for each row that pick_kernel found
//                  too wide (a flat nucleus, a low min-p): histograms of mass.  Launched where the limits
//                  allow such rows
//   rest_kernel    those rows: the cut's bin is gathered and sorted, the slice that u falls into read
//                  again; and what is left (a top-k of nearly 2,048 and more, or of more than there are groups,
//                  infinities, many equals at a wide cut), with sample_row() (sample_select.cuh)
// Vocabularies of more than 2^19 and of less than 16 are sample_row()'s alone.  sample_row() is either all of
// what a kernel does or inlined: as a function that pick_kernel called it gave that kernel a stack, with which a
// launch took 20 us and without which it took 6.  Where no row can be wide and the rows are no more than the
// CUs, pick_kernel has it inlined and rest_kernel is not launched (one row of 50,021: 15.5 to 14.2 us).
//
// Measured, in us (bytes at the 4.8 TB/s of a large copy): 256 rows of 131,072 bf16 without limits 26 (14), of
// which the scan 22.5: some 15 vector instructions a value, 3 of them in 64 bits, bound it; 64 rows of 128,256 f32, top-p 0.95 of flat
// rows, 66 to 70 (7): scan 11, pick 13, slices 11, rest 28, launches behind each other; one row, top-k 50, 14.2, two
// launches.
#include <math.h>

#include <algorithm>
#include <array>
#include <type_traits>

#include "../dtypes.hpp"
#include "kv_common.cuh"
#include "sample_launch.hpp"
#include "sample_select.cuh"

namespace nve_amd {

namespace {

using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;

constexpr int kCandidates = 2 * kThreads;  // sorted at most
constexpr int kCounted = 256;              // placed by counting at most: 64 cost 0.5 us, sorting them 3.7
constexpr int kMostGroups = 8192;
constexpr int kMostUnits = 512;
constexpr int kPieces = 4;               // 16-byte pieces of a lane in a unit
constexpr int kMostSlices = 8;           // of a wide row
// Of a launch: 32 MiB, enough workgroups with one slice a row where there are many rows (up to 8 slices for each of them
// took 2,048 rows of 16,384 f32, top-p 0.95, from 250 to 320 us, 300 of 32,003 bf16 from 84 to 88, and 268 MB).
constexpr int64_t kMostHistograms = 2048;
constexpr int64_t kLeastVocab = 16, kMostVocab = 1 << 19;  // of these kernels: a piece; 8192 groups, 512 units

// A row that pick_kernel left.
struct Wide {
  int32_t kind;             // 0: none; 1: a nucleus; 2: every weight of min_p and more; 3: for sample_row()
  float top, least;         // the greatest value; one below the cut
  unsigned long long target;  // the nucleus' mass times 2^shift
};

// What the kernels leave for the ones behind them, of the rows of a launch.
struct Left {
  int64_t groups, units;
  int32_t group;      // values
  int32_t slices, slice_units;
  float* group_top;   // [rows, groups]
  float* unit_top;    // [rows, units]
  double* unit_mass;  // [rows, units], relative to the unit's maximum
  Wide* wide;         // [rows]
  unsigned long long* bins;  // [rows, slices, kBins]
};

// A row's limits.
struct Limits {
  bool greedy, k_on, p_on, low_on;
  bool plain;  // the temperature leaves everything in f32's range
  int64_t k;
  double p, low, scale, inverse;  // scale: log2(e) / T; inverse: of that
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
    plain = t >= 1e-30f && t <= 1e30f;
    scale = greedy ? 0.0 : 1.4426950408889634 / (double)t;
    inverse = (double)t * 0.6931471805599453;
  }
  __device__ __forceinline__ bool all_mass() const { return !greedy && plain && !k_on && (p_on || !low_on); }
};

// ---------------------------------------------------------------------------
// 2^z in 64 bits
// ---------------------------------------------------------------------------
constexpr int kStepBits = 8;
constexpr int kSteps = 1 << kStepBits;  // of the table

// 2^(j / kSteps) from the exponential's series, with j taken off the exponent's field again, so that
// adding the whole exponent (in units of 1 / kSteps) to the high word gives the power.
constexpr std::array<uint64_t, kSteps> make_powers() {
  std::array<uint64_t, kSteps> t{};
  for (int j = 0; j < kSteps; ++j) {
    const long double x = 0.693147180559945309417232121458L * j / kSteps;
    long double term = 1, sum = 1;
    for (int n = 1; n < 30; ++n) {
      term *= x / n;
      sum += term;
    }
    // 1 <= sum < 2: its 52 bits behind the point
    uint64_t bits = 0;
    long double rest = sum - 1;
    for (int b = 0; b < 52; ++b) {
      rest *= 2;
      bits <<= 1;
      if (rest >= 1) {
        bits |= 1;
        rest -= 1;
      }
    }
    if (rest >= 0.5L) ++bits;
    t[j] = (bits | (uint64_t)1023 << 52) - ((uint64_t)j << (52 - kStepBits));
  }
  return t;
}
__constant__ const std::array<uint64_t, kSteps> kPowers = make_powers();

// A table's power with n, in steps, added to its exponent.
__device__ __forceinline__ double raised(uint64_t power, int n) {
  return __hiloint2double((int)(power >> 32) + (n << (20 - kStepBits)), (int)power);
}

// 2^(steps / kSteps) as a power and the factor that completes it: n, the whole steps, the table, and the series up
// to the third power for the rest, |r| <= 1/2 of a step, whose next term is (ln 2 / 512)^4 / 24 = 1.4e-13.
// near: steps plus 0x1.8p52, which rounds to a whole number; rest: steps plus what it is given, rounded once.
template <typename REST>
__device__ __forceinline__ void power_parts(const uint64_t* table, double near, REST rest, double& power, double& factor) {
  constexpr double k1 = 0.6931471805599453 / kSteps, k2 = k1 * k1 / 2, k3 = k1 * k1 * k1 / 6;
  const int n = (int)__double_as_longlong(near);
  const double r = rest(0x1.8p52 - near);
  double y;  // the compiler would copy k2 for every use
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(y) : "v"(r), "s"(k3), "v"(k2));
  factor = fma(r, fma(r, y, k1), 1.0);
  power = raised(table[n & (kSteps - 1)], n);
}

// Weights 2^((x - high) scale) for x <= high.  Less than 2^-1000 is 0 (parts(): 2^-1000, nothing beside a sum of 1
// and more).
struct Weights {
  const uint64_t* table;
  double high, scale;  // of a step
  double least;        // x - high: what is below has no weight
  __device__ __forceinline__ Weights(const uint64_t* table, const Limits& limits, float high)
      : table(table), high(high), scale(limits.scale * kSteps), least(-1000.0 * limits.inverse) {}
  static __device__ __forceinline__ void fill(uint64_t* t) {
    if (threadIdx.x < kSteps) t[threadIdx.x] = kPowers[threadIdx.x];
  }
  // The power and the factor that completes it; a NaN counts as nothing.
  __device__ __forceinline__ void parts(float x, double& power, double& factor) const {
    const double d = __builtin_fmax((double)x - high, least);
    power_parts(table, fma(d, scale, 0x1.8p52), [&](double more) { return fma(d, scale, more); }, power, factor);
  }
  __device__ __forceinline__ double operator()(float x) const {
    double power, factor;
    parts(x, power, factor);
    return (double)x - high >= least ? power * factor : 0.0;
  }
};

// Adds weights of 16-bit logits, none of them a NaN, to a sum, with what is small in 32 bits, as 64 take twice as long.
// x scale, not (x - high) scale, is taken apart: a difference in 32 bits is 2^-25 of itself off where x is far smaller
// than high.  Whole powers of two of high go with the rounding, and the rest of them is one factor of the sum.
// A weight is within 2^-31 = 4.7e-10 of its value.  In steps, z = x scale < 2^19, with the scale in two floats: what is left
// of z behind its whole steps, r < 0.532, rounds twice, 2^-26 and 2^-25, and misses 2^-29 of z: 1.3e-10 of the weight.
// The series without its 1 has 3/16 of its third power, as a multiple of r, with the first: with the constants'
// rounding 1.3e-10 off; it rounds by 0.532 2^-33 and 2^-34, 1.2e-10.  (1,024 steps, 2^-33: 256 rows of 131,072
// bf16 in 32.6 us in place of 29.6.)
struct Weights16 {
  const uint64_t* table;
  float scale, scale_rest, least;
  float near;  // rounds to a whole number of steps, and takes high's whole powers of two off
  double factor;
  static __device__ __forceinline__ bool fits(const Limits& limits, float high) {
    return fabs((double)high) * limits.scale <= 1024.0;
  }
  __device__ __forceinline__ Weights16(const uint64_t* table, const Limits& limits, float high)
      : table(table), scale((float)(limits.scale * kSteps)), scale_rest((float)(limits.scale * kSteps - (double)scale)),
        least((float)((double)high - 1000.0 * limits.inverse)) {
    const double powers = rint((double)high * limits.scale);
    near = 0x1.8p23f - (float)powers * kSteps;  // exact
    const double steps = fma((double)high, -limits.scale, powers) * kSteps;
    double power, rest;
    power_parts(table, steps + 0x1.8p52, [&](double more) { return steps + more; }, power, rest);
    factor = power * rest;
  }
  // The sum is to be multiplied by the factor.
  __device__ __forceinline__ void add(float x, double& sum) const {
    constexpr double k = 0.6931471805599453 / kSteps;
    constexpr float k1 = (float)(k + 3.0 / 16 * (k * k * k / 6)), k2 = (float)(k * k / 2);
    float y;  // fmaxf() would first make NaNs quiet
    asm("v_max_f32 %0, %1, %2" : "=v"(y) : "v"(x), "v"(least));
    const float t = fmaf(y, scale, near);
    const float r = fmaf(y, scale_rest, fmaf(y, scale, near - t));
    const float more = r * fmaf(r, k2, k1);
    const int n = __float_as_int(t) - __float_as_int(0x1.8p23f);
    const double power = raised(table[n & (kSteps - 1)], n);
    sum = fma(power, (double)more, sum + power);
  }
};

// A lane's 16 bytes of a row (of 16 bytes at least) from `first` on; what is past the row's end is minus infinity.
template <int DT>
struct Piece {
  static constexpr int kValues = 16 / value_elem_bytes(DT);
  u32x4 w;
  // The row's last 16 bytes where those from `first` on would be past its end; settle() then moves them.
  __device__ __forceinline__ void request(const kv_elem<DT>* row, int first, int n) {
    typedef u32x4 __attribute__((aligned(2))) any;  // a row may start at any element
    const uint32_t offset = (uint32_t)min(first, n - kValues) * (uint32_t)sizeof(kv_elem<DT>);
    w = *reinterpret_cast<const any*>(reinterpret_cast<const uint8_t*>(row) + offset);
  }
  __device__ __forceinline__ void settle(int first, int n) {
    if (first + kValues <= n) return;
    constexpr uint64_t kNone = DT == kF32 ? 0xff800000ff800000u : DT == kBF16 ? 0xff80ff80ff80ff80u : 0xfc00fc00fc00fc00u;
    uint64_t x[2];
    __builtin_memcpy(x, &w, 16);
    const int bits = min(kValues, first + kValues - n) * (int)(8 * sizeof(kv_elem<DT>));
    if (bits >= 64) {
      x[0] = x[1];
      x[1] = kNone;
    }
    if (bits == 128) x[0] = kNone;
    if (const int b = bits & 63) {
      x[0] = x[0] >> b | x[1] << (64 - b);
      x[1] = x[1] >> b | kNone << (64 - b);
    }
    __builtin_memcpy(&w, x, 16);
  }
  __device__ __forceinline__ void load(const kv_elem<DT>* row, int first, int n) {
    request(row, first, n);
    settle(first, n);
  }
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (DT == kF32) return __uint_as_float(w[i]);
    if constexpr (DT == kBF16) return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i / 2] >> (i & 1 ? 16 : 0)));
  }
  // The greatest value, or a NaN where there is one among them: this instruction passes on every NaN.  (A maximum of
  // three as max(max(a, b), c) drops a and b where one of them is a signalling NaN, which leaves max(a, b) a quiet one.)
  __device__ __forceinline__ float top() const {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kValues; i += 2)
      asm("v_maximum3_f32 %0, %0, %1, %2" : "+v"(m) : "v"((*this)[i]), "v"((*this)[i + 1]));
    return m;
  }
  // The same of what is no NaN.
  __device__ __forceinline__ float top_of_numbers() const {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kValues; ++i) m = (*this)[i] > m ? (*this)[i] : m;
    return m;
  }
};

template <int DT>
constexpr int unit_values() {
  return kPieces * 64 * Piece<DT>::kValues;
}

// A wave's unit, this lane's pieces from `first` on.
template <int DT>
__device__ __forceinline__ void load_unit(Piece<DT> (&x)[kPieces], const kv_elem<DT>* row, int first, int n) {
  constexpr int kStep = 64 * Piece<DT>::kValues;
#pragma unroll
  for (int j = 0; j < kPieces; ++j) x[j].request(row, first + j * kStep, n);
  if (__any(first + (kPieces - 1) * kStep + Piece<DT>::kValues > n)) {
#pragma unroll
    for (int j = 0; j < kPieces; ++j) x[j].settle(first + j * kStep, n);
  }
}

// ---------------------------------------------------------------------------
// lanes and workgroups
// ---------------------------------------------------------------------------
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

// x of the lane that CTRL names, 0 where it names none; every lane of the wave is on.
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T moved(T x) {
  uint32_t w[sizeof(T) / 4];
  __builtin_memcpy(w, &x, sizeof(T));
#pragma unroll
  for (size_t i = 0; i < sizeof(T) / 4; ++i) {
    w[i] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w[i], CTRL, ROWS, 0xf, false);
    asm volatile("" : "+v"(w[i]));  // not moved under a condition, where some lanes are off
  }
  __builtin_memcpy(&x, w, sizeof(T));
  return x;
}
// Running sums in each row of 16 lanes, and over the wave.
template <typename T>
__device__ __forceinline__ T row_scan(T x) {
  x += moved<0x111, 0xf>(x);
  x += moved<0x112, 0xf>(x);
  x += moved<0x114, 0xf>(x);
  x += moved<0x118, 0xf>(x);
  return x;
}
template <typename T>
__device__ __forceinline__ T lanes_scan(T x) {
  x = row_scan(x);
  x += moved<0x142, 0xa>(x);
  x += moved<0x143, 0xc>(x);
  return x;
}
// x of one lane, the same for all.
template <typename T>
__device__ __forceinline__ T of_lane(T x, int lane) {
  uint32_t w[sizeof(T) / 4];
  __builtin_memcpy(w, &x, sizeof(T));
#pragma unroll
  for (size_t i = 0; i < sizeof(T) / 4; ++i) w[i] = (uint32_t)__builtin_amdgcn_readlane((int)w[i], lane);
  __builtin_memcpy(&x, w, sizeof(T));
  return x;
}

// The sum over 4, 8 or 16 neighbouring lanes.
template <typename T>
__device__ __forceinline__ T group_sum(T x, int bits) {
  x += moved<0xb1, 0xf>(x);
  x += moved<0x4e, 0xf>(x);
  if (bits >= 3) x += moved<0x141, 0xf>(x);
  if (bits >= 4) x += moved<0x140, 0xf>(x);
  return x;
}

// x of the threads up to and including this one, added in one order; total: of all.
template <typename T>
__device__ __forceinline__ T block_scan(T x, T* red, T& total) {
  static_assert(kWaves == 16);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  x = lanes_scan(x);
  __syncthreads();
  if (lane == 63) red[wave] = x;
  __syncthreads();
  const T r = row_scan(red[lane & 15]);
  total = of_lane(r, 15);
  if (wave > 0) x += of_lane(r, wave - 1);
  return x;
}

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

// Sorts n <= kCandidates keys, the greatest first; those behind them up to a power of two become 0.
__device__ __forceinline__ void sort_keys(uint64_t* keys, int n) {
  const int tid = threadIdx.x;
  int size2 = 2;
  while (size2 < n) size2 <<= 1;
  for (int i = n + tid; i < size2; i += kThreads) keys[i] = 0;
  __syncthreads();
  const bool one_wave = size2 <= 128;
  if (!one_wave || tid < 64) {
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
        if (one_wave) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        else __syncthreads();
      }
    }
  }
  __syncthreads();
}

// kBins bins of one width from `high` down; the first one has all that is above (and what is no number), the last one
// all that is below.  A width past f32 leaves a scale that keeps the order.
struct Steps {
  float high, scale;
  __device__ __forceinline__ Steps(float high, float low) : high(high) {
    const float width = high - low;
    scale = width > 0.0f ? fminf(fmaxf((kBins - 0.1f) / width, 1e-36f), 3e38f) : 3e38f;
  }
  __device__ __forceinline__ int of(float x) const {
    return (int)__builtin_amdgcn_fmed3f((high - x) * scale, 0.0f, kBins - 1.0f);
  }
  // Values above all and below all of bin b's: a bin's width and 2^-20 away, more than any rounding; or NaN.
  __device__ __forceinline__ float above(int b) const { return away((float)(b - 1), 0x1p-20f); }
  __device__ __forceinline__ float below(int b) const { return b == kBins - 1 ? -INFINITY : away((float)(b + 2), -0x1p-20f); }
  __device__ __forceinline__ float away(float bins, float more) const {
    const float edge = high - bins / scale;
    return edge + (fabsf(high) + fabsf(edge)) * more;
  }
};

// ---------------------------------------------------------------------------
// the first kernel: a unit a wave
// ---------------------------------------------------------------------------
constexpr int kScanThreads = 256;

// More units a wave, the next one's pieces requested as this one's are summed, took longer (256 rows of 131,072 bf16:
// 1 unit 22.8 us, 2 23.6, 4 25.1; f32 32.6, 37.2, 36.9).
template <int DT, int GROUP>
__global__ __launch_bounds__(kScanThreads, 7) void scan_kernel(const Sample a, const Left l, const int blocks) {
  constexpr int kValues = Piece<DT>::kValues, kLanes = GROUP / kValues, kUnit = unit_values<DT>();
  __shared__ uint64_t table[kSteps];
  const int lane = threadIdx.x & 63, vocab = (int)a.vocab;
  const int64_t row = blockIdx.x / blocks;
  const int unit = __builtin_amdgcn_readfirstlane((int)(blockIdx.x - row * blocks) * (kScanThreads / 64) +
                                                  (int)(threadIdx.x >> 6));
  const int base = unit * kUnit + lane * kValues;
  Piece<DT> x[kPieces];
  load_unit(x, reinterpret_cast<const kv_elem<DT>*>(a.logits) + row * a.row_stride, base, vocab);
  const Limits limits(a, row);
  const bool sums = limits.all_mass();
  if (sums) Weights::fill(table);
  __syncthreads();
  if (unit >= (int)l.units) return;
  float tops[kPieces];
  bool odd = false;
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    tops[j] = x[j].top();
    odd |= tops[j] != tops[j];
  }
  const bool nans = __any(odd);
  if (nans) {
#pragma unroll
    for (int j = 0; j < kPieces; ++j) tops[j] = x[j].top_of_numbers();
  }
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    const float m = lanes_max<kLanes>(tops[j]);
    const int group = (base + j * 64 * kValues) / GROUP;
    if (lane % kLanes == 0 && group < (int)l.groups) l.group_top[row * l.groups + group] = m;
    top = fmaxf(top, m);
  }
  if (!sums) return;
  top = lanes_max<64>(top);
  double sum = 0.0;
  if (top > -INFINITY && top < INFINITY) {
    // piece by piece: all values taken apart together, as for the maxima, would need too many registers
    auto add = [&](auto one) {
#pragma unroll
      for (int j = 0; j < kPieces; ++j) {
        asm volatile("" : "+v"(x[j].w));
#pragma unroll
        for (int i = 0; i < kValues; ++i) one(x[j][i]);
        asm volatile("" : "+v"(sum));
      }
      sum = of_lane(lanes_scan(sum), 63);
    };
    auto exact = [&] {
      const Weights weights(table, limits, top);
      add([&](float v) {
        double power, factor;
        weights.parts(v, power, factor);
        sum = fma(power, factor, sum);
      });
    };
    if constexpr (DT == kF32) {
      exact();
    } else if (!nans && __builtin_amdgcn_readfirstlane(Weights16::fits(limits, top))) {
      const Weights16 weights(table, limits, top);
      add([&](float v) { weights.add(v, sum); });
      sum *= weights.factor;
    } else {
      exact();
    }
  }
  if (lane == 0) {
    l.unit_top[row * l.units + unit] = top;
    l.unit_mass[row * l.units + unit] = sum;
  }
}

// ---------------------------------------------------------------------------
// a row in one workgroup
// ---------------------------------------------------------------------------
struct RowShared {
  union {
    float tops[kMostGroups];
    struct {
      uint64_t keys[kCandidates];  // in the vocabulary's order
      uint64_t some[kCandidates];  // those around a cut
    };
  };
  union {
    uint16_t groups[kCandidates];
    unsigned long long mass[kBins];
  };
  uint64_t table[kSteps];
  double part[kMostUnits / kMostSlices * kPieces];
  double red_sum[kWaves];
  unsigned long long red_mass[kWaves];
  int red_count[kWaves];
  float red_low[kWaves], red_high[kWaves];
  unsigned long long slice[kMostSlices], slices[kMostSlices][kWaves];
  int first_item[kWaves], last_item[kWaves], bin, n;
  double first_before[kWaves], last_before[kWaves];
  unsigned long long before_mass;
  uint64_t cut;
};

union AnyShared {
  SelectShared select;
  RowShared row;
};
struct RowSharedAlone {
  RowShared row;
};

template <int DT, int GROUP>
struct Pick {
  static constexpr int kValues = Piece<DT>::kValues, kLanes = GROUP / kValues, kUnit = unit_values<DT>();
  const Sample& a;
  const Left& l;
  const Limits& limits;
  RowShared& s;
  const int64_t row;
  const kv_elem<DT>* p;
  double mass_scale;
  float top;
  double u;

  __device__ __forceinline__ double weight(float x) const { return Weights(s.table, limits, top)(x); }
  // A weight, 1 at most, times 2^shift, 2^51 at most, rounded by adding 2^52; those of a row sum to less than 2^62.
  __device__ __forceinline__ unsigned long long mass_of(double w) const {
    return (unsigned long long)__double_as_longlong(w * mass_scale + 0x1p52) & ((1ull << 52) - 1);
  }
  __device__ __forceinline__ void answer(int64_t token) const {
    if (threadIdx.x == 0) a.tokens[row] = token;
  }

  // The bin at which the running sum of two bins a thread reaches the target, or -1; s.before_mass: before it.
  __device__ __forceinline__ int bin_at(unsigned long long x0, unsigned long long x1, unsigned long long target) const {
    const int tid = threadIdx.x;
    unsigned long long total;
    const unsigned long long end = block_scan<unsigned long long>(x0 + x1, s.red_mass, total);
    if (total < target) return -1;
    const unsigned long long b1 = end - x1, b0 = b1 - x0;
    if (b0 < target && b1 >= target) {
      s.bin = 2 * tid;
      s.before_mass = b0;
    } else if (b1 < target && end >= target) {
      s.bin = 2 * tid + 1;
      s.before_mass = b1;
    }
    __syncthreads();
    return s.bin;
  }

  // The first of the threads' two items each at which the running sum of their weights, from `base` on, exceeds
  // the target; the last one with a weight where none does.  share: the target is that times the sum.
  // before: the running sum before it.
  __device__ __forceinline__ int pick_item(double w0, double w1, double base, double& target, bool share,
                                           double& before) const {
    const int i = 2 * threadIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double total;
    const double end = base + block_scan(w0 + w1, s.red_sum, total);
    if (share) target *= total;
    const bool f0 = w0 > 0.0 && end - w1 > target, f1 = w1 > 0.0 && end > target;
    const uint64_t over = __ballot(f0 || f1), any = __ballot(w0 > 0.0 || w1 > 0.0);
    if (over ? lane == __builtin_ctzll(over) : lane == 0) {
      s.first_item[wave] = over ? (f0 ? i : i + 1) : -1;
      s.first_before[wave] = f0 ? end - w1 - w0 : end - w1;
    }
    if (any ? lane == 63 - __builtin_clzll(any) : lane == 0) {
      s.last_item[wave] = any ? (w1 > 0.0 ? i + 1 : i) : -1;
      s.last_before[wave] = w1 > 0.0 ? end - w1 : end - w1 - w0;
    }
    __syncthreads();
    const uint64_t first = __ballot(s.first_item[lane & 15] >= 0) & 0xffff;
    const uint64_t last = __ballot(s.last_item[lane & 15] >= 0) & 0xffff;
    const int w = first ? __builtin_ctzll(first) : last ? 63 - __builtin_clzll(last) : 0;
    const int item = first ? s.first_item[w] : s.last_item[w];
    before = first ? s.first_before[w] : s.last_before[w];
    __syncthreads();
    return item;
  }

  // Greatest and least of the finite ones of lo and hi over the workgroup.
  __device__ __forceinline__ void reduce_range(float& lo, float& hi) const {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    hi = lanes_max<64>(hi);
    lo = -lanes_max<64>(-lo);
    if (lane == 0) {
      s.red_high[wave] = hi;
      s.red_low[wave] = lo;
    }
    __syncthreads();
    hi = lanes_max<16>(s.red_high[lane & 15]);
    lo = -lanes_max<16>(-s.red_low[lane & 15]);
  }

  // The one of n keys in s.some at which the running sum, in the order, of ones or (by_mass) masses reaches the
  // target; 0 if it never does.
  __device__ __forceinline__ uint64_t place_of(int n, bool by_mass, unsigned long long target) const {
    const int tid = threadIdx.x;
    if (tid == 0) s.cut = 0;
    if (n <= kCounted) {  // what is ahead of each, by comparing it with all: 4 to 16 threads a key
      if (tid < n) s.mass[tid] = by_mass ? mass_of(weight(value_of(s.some[tid]))) : 1;
      __syncthreads();
      const int bits = n <= 64 ? 4 : n <= 128 ? 3 : 2, mine_at = tid >> bits, part = tid & ((1 << bits) - 1);
      unsigned long long ahead = 0;
      if (mine_at < n) {
        const uint64_t key = s.some[mine_at];
        for (int j = part; j < n; j += 1 << bits) ahead += s.some[j] > key ? s.mass[j] : 0;
      }
      ahead = group_sum(ahead, bits);
      if (mine_at < n && part == 0 && ahead < target && ahead + s.mass[mine_at] >= target) s.cut = s.some[mine_at];
    } else {
      sort_keys(s.some, n);
      const int i = 2 * tid;
      unsigned long long m[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) m[j] = i + j >= n ? 0 : by_mass ? mass_of(weight(value_of(s.some[i + j]))) : 1;
      const int j = bin_at(m[0], m[1], target);
      if (tid == 0 && j >= 0) s.cut = s.some[j];
    }
    __syncthreads();
    return s.cut;
  }

  // The same among the n keys in s.keys.
  __device__ __forceinline__ uint64_t cut_of(int n, bool by_mass, unsigned long long target) const {
    const int tid = threadIdx.x;
    if (n <= kCounted) {
      if (tid < n) s.some[tid] = s.keys[tid];
      __syncthreads();
      return place_of(n, by_mass, target);
    }
    // the bin that it is in, then those in the bin
    float v[2], lo = INFINITY, hi = -INFINITY;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = tid + j * kThreads;
      v[j] = i < n ? value_of(s.keys[i]) : 0.0f;
      if (i < n) lo = fminf(lo, v[j]);
      s.mass[i] = 0;
    }
    reduce_range(lo, hi);
    const Steps steps(top, lo);
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (tid + j * kThreads < n) atomicAdd(&s.mass[steps.of(v[j])], by_mass ? mass_of(weight(v[j])) : 1ull);
    if (tid == 0) s.n = 0;
    __syncthreads();
    const int bin = bin_at(s.mass[2 * tid], s.mass[2 * tid + 1], target);
    if (bin < 0) return 0;
    const unsigned long long before = s.before_mass;
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (tid + j * kThreads < n && steps.of(v[j]) == bin) s.some[atomicAdd(&s.n, 1)] = s.keys[tid + j * kThreads];
    __syncthreads();
    return place_of(s.n, by_mass, target - before);
  }

  // The token among `size` values from `first` on, 2,048 at most: those from `cut` on, the least weight `low`.
  __device__ __forceinline__ void pick_in(int64_t first, int size, double base, double target, uint64_t cut, double low) const {
    double w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t at = first + 2 * threadIdx.x + i;
      w[i] = 0.0;
      if (2 * (int)threadIdx.x + i < size && at < a.vocab) {
        const float x = (float)p[at];
        const double y = weight(x);
        if (x > -INFINITY && key_of(x, at) >= cut && y >= low) w[i] = y;
      }
    }
    double before;
    answer(first + pick_item(w[0], w[1], base, target, false, before));
  }

  enum Found { kDone, kWide, kElse };

  __device__ __forceinline__ Found run(Wide& left) {
    const int tid = threadIdx.x;
    if (!limits.greedy && !limits.plain) return kElse;
    Weights::fill(s.table);
    u = a.u[row] > 0.0f ? (double)a.u[row] : 0.0;
    float lo = INFINITY, hi = -INFINITY;

    double all = 0.0;  // the mass of all, where it counts
    if (limits.all_mass()) {
      const int i = 2 * tid;
      float t[2] = {-INFINITY, -INFINITY};
      double m[2] = {0.0, 0.0};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (i + j < l.units) {
          t[j] = l.unit_top[row * l.units + i + j];
          m[j] = l.unit_mass[row * l.units + i + j];
        }
      }
      hi = fmaxf(t[0], t[1]);
      reduce_range(lo, hi);
      top = hi;
      if (top == -INFINITY) {
        answer(-1);
        return kDone;
      }
      if (top == INFINITY) return kElse;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 2; ++j) m[j] = t[j] > -INFINITY ? m[j] * weight(t[j]) : 0.0;
      if (!limits.p_on) {
        double target = u, before;
        const int unit = pick_item(m[0], m[1], 0.0, target, true, before);
        pick_in((int64_t)unit * kUnit, kUnit, before, target, 0, 0.0);
        return kDone;
      }
      block_scan(m[0] + m[1], s.red_sum, all);
      __syncthreads();
      lo = INFINITY;
      hi = -INFINITY;
    }

    for (int64_t g = tid; g < l.groups; g += kThreads) {
      const float t = l.group_top[row * l.groups + g];
      s.tops[g] = t;
      hi = fmaxf(hi, t);
      if (t > -INFINITY) lo = fminf(lo, t);
    }
    reduce_range(lo, hi);
    top = hi;
    if (top == -INFINITY) {
      answer(-1);
      return kDone;
    }
    if (top == INFINITY) return kElse;

    // candidates: values in the first `limit` + 1 steps and not below `least`
    const Steps steps(top, lo);
    int limit = kBins;
    int most = kCandidates;  // groups that are read
    float least = -INFINITY;
    unsigned long long target = 0;
    if (limits.greedy) {
      least = top;
    } else {
      // min-p's tokens are a part of a nucleus or hold all of it, but top-p's sum after top-k is of all of top-k's
      if (limits.low_on && !(limits.k_on && limits.p_on)) {
        // a little below the least weight's value: what is between is left out by its weight
        const double high = top, low = high + log2(limits.low) / limits.scale;
        least = (float)(low - 1e-6 * fabs(low) - 1e-6 * fabs(high));
      }
      target = (unsigned long long)fmax(ceil(limits.p * all * mass_scale), 1.0);
      if ((limits.k_on || limits.p_on) && a.vocab > kCandidates) {
        if (limits.k_on && limits.k > kCandidates) return kElse;
        for (int i = tid; i < kBins; i += kThreads) s.mass[i] = 0;
        __syncthreads();
        for (int64_t g = tid; g < l.groups; g += kThreads) {
          const float t = s.tops[g];
          if (t > -INFINITY) atomicAdd(&s.mass[steps.of(t)], limits.k_on ? 1ull : mass_of(weight(t)));
        }
        __syncthreads();
        if (limits.k_on) {
          limit = bin_at(s.mass[2 * tid], s.mass[2 * tid + 1], limits.k);
          if (limit < 0) return kElse;
        } else {
          const int sure = bin_at(s.mass[2 * tid], s.mass[2 * tid + 1], target);
          if (sure >= 0 || !limits.low_on) {
            // else the maxima that sum to most of it, if they are few: likely with all of it around them (64 rows of
            // 128,256, top-p 0.95: 26 us with up to 2,048 groups, 13 with 512)
            if (sure < 0) most = 512;
            limit = sure >= 0 ? sure : bin_at(s.mass[2 * tid], s.mass[2 * tid + 1], target - target / 4);
            if (limit < 0) limit = kBins;
          }
        }
      }
      // A nucleus leaves out (1 - p) of the mass at most, so its least weight is at least that over the vocabulary.
      float bound = least;
      if (limits.p_on) {
        const double depth = log2((double)a.vocab / ((1.0 - limits.p) * all)) / limits.scale;
        bound = (float)((double)top - fmax(depth, 0.0) * 1.0001 - 1e-6 * fabs((double)top));
      }
      left = Wide{limits.p_on ? 1 : 2, top, bound, target};
    }
    const Found rest = !limits.k_on && left.least > -3e38f ? kWide : kElse;
    auto wanted = [&](float x) { return x >= least && x > -INFINITY && (limit >= kBins || steps.of(x) <= limit); };

    // the groups with candidates, in order
    const int per = (int)((l.groups + kThreads - 1) / kThreads), g0 = tid * per;
    uint32_t mine = 0;
    for (int i = 0; i < per; ++i) mine |= (uint32_t)(g0 + i < l.groups && wanted(s.tops[g0 + i])) << i;
    int groups;
    int at = block_scan((int)__popc(mine), s.red_count, groups) - __popc(mine);
    bool few = groups <= most;
    int n = 0;
    if (few) {
      for (; mine; mine &= mine - 1) s.groups[at++] = (uint16_t)(g0 + __builtin_ctz(mine));
      __syncthreads();
      // their candidates, in order: four groups a lane group in a round
      constexpr int kStep = kThreads / kLanes;
      for (bool again = limits.k_on;; again = false) {
        for (int b0 = 0; b0 < groups && few; b0 += 4 * kStep) {
          Piece<DT> x[4];
          uint32_t yes[4];
          unsigned long long counts = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int mine_at = b0 + j * kStep + tid / kLanes;
            yes[j] = 0;
            if (mine_at < groups) x[j].load(p, s.groups[mine_at] * GROUP + tid % kLanes * kValues, (int)a.vocab);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int mine_at = b0 + j * kStep + tid / kLanes;
            if (mine_at < groups) {
#pragma unroll
              for (int i = 0; i < kValues; ++i) yes[j] |= (uint32_t)wanted(x[j][i]) << i;
            }
            counts |= (unsigned long long)__popc(yes[j]) << (16 * j);
          }
          unsigned long long more;
          const unsigned long long before = block_scan(counts, s.red_mass, more) - counts;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int count = (int)(more >> (16 * j)) & 0xffff;
            few = few && n + count <= kCandidates;
            if (few && yes[j]) {
              int to = n + ((int)(before >> (16 * j)) & 0xffff);
              const int64_t first = (int64_t)s.groups[b0 + j * kStep + tid / kLanes] * GROUP + tid % kLanes * kValues;
#pragma unroll
              for (int i = 0; i < kValues; ++i)
                if (yes[j] >> i & 1) s.keys[to++] = key_of(x[j][i], first + i);
            }
            n += count;
          }
        }
        if (few || !again) break;
        // Too many for top-k: groups above the k-th maximum hold more tokens above it.  The step that the k-th token
        // itself is in leaves few more than k (64 rows of 32,003 f16, top-k 2,000: 102 us by sample_row(), so 29; of
        // 128,256 f32 327 and 64).
        __syncthreads();
        auto* counts = reinterpret_cast<unsigned long long*>(s.some);
        static_assert(sizeof(s.some) == kBins * sizeof(unsigned long long));
        for (int i = tid; i < kBins; i += kThreads) counts[i] = 0;
        __syncthreads();
        for (int b0 = tid / kLanes; b0 < groups; b0 += kStep) {
          Piece<DT> x;
          x.load(p, s.groups[b0] * GROUP + tid % kLanes * kValues, (int)a.vocab);
#pragma unroll
          for (int i = 0; i < kValues; ++i)
            if (wanted(x[i])) atomicAdd(&counts[steps.of(x[i])], 1ull);
        }
        __syncthreads();
        limit = bin_at(counts[2 * tid], counts[2 * tid + 1], limits.k);
        if (limit < 0) return kElse;
        n = 0;
        few = true;
      }
    }
    __syncthreads();
    if (limits.greedy) {  // the first of them
      if (few) answer(index_of(s.keys[0]));
      return few ? kDone : kElse;
    }
    if (!few) return rest;

    uint64_t cut = 0;
    const int i = 2 * tid;
    if (limits.k_on && n > limits.k) cut = cut_of(n, false, limits.k);
    double w[2] = {0.0, 0.0};
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (i + j < n && s.keys[i + j] >= cut) w[j] = weight(value_of(s.keys[i + j]));
    if (limits.p_on) {
      unsigned long long total;
      block_scan<unsigned long long>(mass_of(w[0]) + mass_of(w[1]), s.red_mass, total);
      if (limits.k_on) target = (unsigned long long)fmax(ceil(limits.p * (double)total), 1.0);
      if (total >= target) {
        cut = max(cut, cut_of(n, true, target));
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (i + j < n && s.keys[i + j] < cut) w[j] = 0.0;
      } else if (!limits.low_on && a.vocab > kCandidates) {
        return rest;  // the candidates are not all of the nucleus
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (w[j] < limits.low) w[j] = 0.0;
    double share = u, before;
    answer(index_of(s.keys[pick_item(w[0], w[1], 0.0, share, true, before)]));
    return kDone;
  }

  // A wide row from its slices' histograms; false: not decided here.
  __device__ __forceinline__ bool finish(const Wide& of) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    Weights::fill(s.table);
    u = a.u[row] > 0.0f ? (double)a.u[row] : 0.0;
    top = of.top;
    const Steps steps(top, of.least);
    const unsigned long long* bins = l.bins + row * l.slices * kBins;
    int whole = kBins;  // bins before it are kept whole
    uint64_t cut = 0;
    int n = 0;
    unsigned long long x[kMostSlices][2];
#pragma unroll
    for (int j = 0; j < kMostSlices; ++j) {
      x[j][0] = j < l.slices ? bins[j * kBins + 2 * tid] : 0;
      x[j][1] = j < l.slices ? bins[j * kBins + 2 * tid + 1] : 0;
    }
    if (of.kind == 1) {
      unsigned long long x0 = 0, x1 = 0;
#pragma unroll
      for (int j = 0; j < kMostSlices; ++j) {
        x0 += x[j][0];
        x1 += x[j][1];
      }
      const int bin = bin_at(x0, x1, of.target);
      if (bin < 0) return false;
      // the bins that need a look at their values: the nucleus' last one, or those around min-p's value where
      // that comes first
      int last = bin;
      whole = bin;
      if (limits.low_on) {
        const int low = steps.of((float)((double)top + log2(limits.low) / limits.scale));
        whole = min(bin, max(low - 1, 0));
        last = min(bin, low + 1);
      }
      unsigned long long above;
      block_scan((2 * tid < whole ? x0 : 0) + (2 * tid + 1 < whole ? x1 : 0), s.red_mass, above);
      if (tid == 0) s.n = 0;
      __syncthreads();
      // two comparisons before the bin, which takes some more instructions (a NaN above passes); with the runs below in
      // place of units 100 rows of 32,003 f16 took 49.6 us a call, 52.8 without, 64 of 128,256 f32 67.5 and 68.6
      const float above_all = steps.above(whole), below_all = fmaxf(steps.below(last), of.least);
      constexpr int kAhead = 2;  // units whose loads are under way together
      for (int64_t unit = wave; unit < l.units; unit += kAhead * kWaves) {
        Piece<DT> y[kAhead][kPieces];
#pragma unroll
        for (int h = 0; h < kAhead; ++h) load_unit(y[h], p, (int)((unit + h * kWaves) * kUnit) + lane * kValues, (int)a.vocab);
#pragma unroll
        for (int h = 0; h < kAhead; ++h) {
          if (unit + h * kWaves >= l.units) break;
#pragma unroll
          for (int j = 0; j < kPieces; ++j) {
            bool some = false;
#pragma unroll
            for (int i = 0; i < kValues; ++i) some |= (int)!(y[h][j][i] > above_all) & (int)(y[h][j][i] >= below_all);
            if (!some) continue;
#pragma unroll
            for (int i = 0; i < kValues; ++i) {
              const int b = steps.of(y[h][j][i]);
              if (b >= whole && b <= last && y[h][j][i] >= of.least) {
                const int at = atomicAdd(&s.n, 1);
                if (at < kCandidates)
                  s.some[at] = key_of(y[h][j][i], (unit + h * kWaves) * kUnit + (j * 64 + lane) * kValues + i);
              }
            }
          }
        }
      }
      __syncthreads();
      n = s.n;
      if (n > kCandidates) return false;
      cut = place_of(n, true, of.target > above ? of.target - above : 1);
      if (cut == 0 && last == bin) return false;
    }
    // the slices' kept masses
#pragma unroll
    for (int j = 0; j < kMostSlices; ++j) {
      unsigned long long sum = (2 * tid < whole ? x[j][0] : 0) + (2 * tid + 1 < whole ? x[j][1] : 0);
      sum = lanes_scan(sum);
      if (lane == 63) s.slices[j][wave] = sum;
    }
    __syncthreads();
    if (wave < l.slices) {
      unsigned long long sum = lane < kWaves ? s.slices[wave][lane] : 0;
      for (int j = lane; j < n; j += 64) {
        const uint64_t key = s.some[j];
        const double w = weight(value_of(key));
        if (key >= cut && w >= limits.low && index_of(key) / (kUnit * l.slice_units) == wave) sum += mass_of(w);
      }
      sum = of_lane(lanes_scan(sum), 63);
      if (lane == 0) s.slice[wave] = sum;
    }
    __syncthreads();
    unsigned long long total = 0;
    for (int j = 0; j < l.slices; ++j) total += s.slice[j];
    const double target = u * ((double)total / mass_scale);
    int slice = -1;
    double base = 0.0;
    unsigned long long sum = 0;
    for (int j = 0; j < l.slices; ++j) {
      if (s.slice[j] == 0) continue;
      slice = j;
      base = (double)sum / mass_scale;
      sum += s.slice[j];
      if ((double)sum / mass_scale > target) break;
    }
    if (slice < 0) return false;
    // the runs' of a wave's piece in that slice
    const Weights weights(s.table, limits, top);
    const float cut_value = cut ? value_of(cut) : -INFINITY;
    const int64_t cut_index = cut ? index_of(cut) : -1;
    const int64_t first = (int64_t)slice * l.slice_units, last = min(first + l.slice_units, l.units);
    constexpr int kPart = 64 * kValues;
    const int64_t part0 = first * kPieces, count = (last - first) * kPieces;
    for (int at0 = wave; at0 < count; at0 += 4 * kWaves) {
      Piece<DT> x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j].load(p, (int)(part0 + at0 + j * kWaves) * kPart + lane * kValues, (int)a.vocab);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (at0 + j * kWaves >= count) break;
        const int64_t at = (part0 + at0 + j * kWaves) * kPart + lane * kValues;
        double mass = 0.0;
#pragma unroll
        for (int i = 0; i < kValues; ++i) {
          const float v = x[j][i];
          const double w = weights(v);
          const bool kept = (v > cut_value || (v == cut_value && at + i <= cut_index)) && w >= limits.low;
          mass += kept ? w : 0.0;
        }
        mass = of_lane(lanes_scan(mass), 63);
        if (lane == 0) s.part[at0 + j * kWaves] = mass;
      }
    }
    __syncthreads();
    const int i = 2 * tid;
    double to = target;
    double before;
    const int part = pick_item(i < count ? s.part[i] : 0.0, i + 1 < count ? s.part[i + 1] : 0.0, base, to, false, before);
    pick_in((part0 + part) * kPart, kPart, before, to, cut, limits.low);
    return true;
  }
};

// ALONE: nothing is left for rest_kernel, which is not launched.
template <int DT, int GROUP, bool ALONE>
__global__ __launch_bounds__(kThreads) void pick_kernel(const Sample a, const Left l, const int shift) {
  __shared__ std::conditional_t<ALONE, AnyShared, RowSharedAlone> s;
  const int64_t row = blockIdx.x;
  const Limits limits(a, row);
  using P = Pick<DT, GROUP>;
  P pick{a, l, limits, s.row, row, reinterpret_cast<const kv_elem<DT>*>(a.logits) + row * a.row_stride,
         __hiloint2double((1023 + shift) << 20, 0)};
  Wide left{};
  const typename P::Found found = pick.run(left);
  if constexpr (ALONE) {
    if (found == P::kDone) return;
    __syncthreads();
    sample_row<DT>(a, shift, row, s.select);
  } else if (threadIdx.x == 0) {
    if (found == P::kDone) left.kind = 0;
    else if (found == P::kElse || l.slices == 0) left.kind = 3;
    l.wide[row] = left;
  }
}

// Masses of a slice's values in bins.
constexpr int kSliceThreads = 512;

template <int DT>
__global__ __launch_bounds__(kSliceThreads) void slice_kernel(const Sample a, const Left l, const int shift) {
  constexpr int kValues = Piece<DT>::kValues, kUnit = unit_values<DT>();
  __shared__ unsigned long long mass[kBins];
  __shared__ uint64_t table[kSteps];
  const int64_t row = blockIdx.x / l.slices;
  const int slice = blockIdx.x - row * l.slices;
  const Wide of = l.wide[row];
  if (of.kind != 1 && of.kind != 2) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int i = threadIdx.x; i < kBins; i += kSliceThreads) mass[i] = 0;
  Weights::fill(table);
  __syncthreads();
  const Limits limits(a, row);
  const Weights weights(table, limits, of.top);
  const Steps steps(of.top, of.least);
  const double mass_scale = __hiloint2double((1023 + shift) << 20, 0);
  const double low = of.kind == 2 ? limits.low : 0.0;
  const kv_elem<DT>* p = reinterpret_cast<const kv_elem<DT>*>(a.logits) + row * a.row_stride;
  const int64_t last = min((int64_t)(slice + 1) * l.slice_units, l.units);
  for (int64_t unit = (int64_t)slice * l.slice_units + wave; unit < last; unit += kSliceThreads / 64) {
    const int64_t base = unit * kUnit + lane * kValues;
    Piece<DT> x[kPieces];
    load_unit(x, p, (int)base, (int)a.vocab);
#pragma unroll
    for (int j = 0; j < kPieces; ++j)
#pragma unroll
      for (int i = 0; i < kValues; ++i) {
        if (x[j][i] >= of.least) {
          const double w = weights(x[j][i]);
          if (w >= low)
            atomicAdd(&mass[steps.of(x[j][i])],
                      (unsigned long long)__double_as_longlong(w * mass_scale + 0x1p52) & ((1ull << 52) - 1));
        }
      }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += kSliceThreads) l.bins[(row * l.slices + slice) * kBins + i] = mass[i];
}

// What pick_kernel left.
template <int DT>
__global__ __launch_bounds__(kThreads) void rest_kernel(const Sample a, const Left l, const int shift) {
  __shared__ AnyShared s;
  const int64_t row = blockIdx.x;
  const Wide of = l.wide[row];
  if (of.kind == 0) return;
  if (of.kind < 3) {
    const Limits limits(a, row);
    Pick<DT, 64> pick{a, l, limits, s.row, row, reinterpret_cast<const kv_elem<DT>*>(a.logits) + row * a.row_stride,
                      __hiloint2double((1023 + shift) << 20, 0)};
    if (pick.finish(of)) return;
    __syncthreads();
  }
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

// Rows of a launch: 2^25 values, but some hundred rows at least, whose workspace the next launch takes over.
int64_t most_rows(const Sample& a) {
  return std::min(a.rows, std::max<int64_t>(256, ((int64_t)1 << 25) / std::max<int64_t>(a.vocab, 1 << 14)));
}

// Whether scan_kernel and pick_kernel take the rows.
bool in_kernels(const Sample& a) { return a.vocab >= kLeastVocab && a.vocab <= kMostVocab; }

int unit_of(int dtype) { return dtype == kF32 ? unit_values<kF32>() : unit_values<kF16>(); }

// Whether a row may keep more tokens than pick_kernel sorts, as far as the host can see.
bool may_be_wide(const Sample& a) {
  if (a.vocab <= kCandidates) return false;
  if (!a.temperature && a.temperature_all == 0.0f) return false;
  if (!a.top_k && a.top_k_all > 0 && a.top_k_all < a.vocab) return false;
  return a.top_p || a.top_p_all < 1.0f || a.min_p || a.min_p_all > 0.0f;
}

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
  if (may_be_wide(a)) {
    const int64_t slices = std::max<int64_t>(1, std::min<int64_t>(kMostSlices, kMostHistograms / (int64_t)rows));
    l.slice_units = (int)((l.units + slices - 1) / slices);
    l.slices = (int)((l.units + l.slice_units - 1) / l.slice_units);
    l.bins = static_cast<unsigned long long*>(take(rows * l.slices * kBins * 8));
  }
  l.wide = static_cast<Wide*>(take(rows * sizeof(Wide)));
  *bytes = used;
  return l;
}

template <int DT, int GROUP>
void launch_groups(const Sample& a, const Left& l, int shift, hipStream_t stream) {
  const unsigned n = (unsigned)a.rows;
  const int blocks = (int)((l.units + kScanThreads / 64 - 1) / (kScanThreads / 64));
  scan_kernel<DT, GROUP><<<n * blocks, kScanThreads, 0, stream>>>(a, l, blocks);
  // sample_row()'s registers leave one workgroup a CU; a launch without rows to do takes 1.5 us and more
  if (l.slices == 0 && a.rows <= 256) {
    pick_kernel<DT, GROUP, true><<<n, kThreads, 0, stream>>>(a, l, shift);
    return;
  }
  pick_kernel<DT, GROUP, false><<<n, kThreads, 0, stream>>>(a, l, shift);
  if (l.slices > 0) slice_kernel<DT><<<n * l.slices, kSliceThreads, 0, stream>>>(a, l, shift);
  rest_kernel<DT><<<n, kThreads, 0, stream>>>(a, l, shift);
}

template <int DT>
hipError_t launch_rows(const Sample& a, const Left& l, int shift, hipStream_t stream) {
  if (!in_kernels(a)) select_kernel<DT><<<(unsigned)a.rows, kThreads, 0, stream>>>(a, shift);
  else if (l.group == 16) launch_groups<DT, 16>(a, l, shift, stream);
  else launch_groups<DT, 64>(a, l, shift, stream);
  return hipGetLastError();
}

}  // namespace

size_t sample_workspace(const Sample& a) {
  size_t bytes = 0;
  if (a.rows > 0 && in_kernels(a)) layout_of(a, nullptr, &bytes);
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
