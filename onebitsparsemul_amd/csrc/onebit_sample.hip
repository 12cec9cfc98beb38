// Tokens from logits (onebit_head.h). Nothing is sorted: the filters keep what lies above a value, and of the logits equal to it those of the lowest indices, so
// that each of them is a search for that value, digit by digit from the top in a histogram of counts and masses. Masses are integers (2^-42 of the largest
// weight): their sums do not depend on an order, and 2^-43 is the most a weight is off, so that which token a number falls on is what 64-bit sums give.
#include "onebit_decoder_device.h"
#include "onebit_head_launch.h"

namespace onebit {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = 2048, kFraction = 42;
typedef unsigned long long mass_t;

// Floats as integers of the same order; -0 as 0.
__device__ inline uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ inline float value_of(uint32_t key) { return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xffffffffu)); }
constexpr uint32_t kKeyOfMinusInfinity = 0x007fffffu;

// The weight of a logit as an integer: 2^(distance + 42), distance = log2 e (logit - largest) / temperature <= 0. 2^n r, r by the exponential series of the fraction
// of n, at most 1/2: its twelve terms leave 2e-14 out.
__device__ inline mass_t weight_of(double distance) {
  if (!(distance >= -kFraction - 1)) return 0;
  const double n = __builtin_rint(distance), x = (distance - n) * 0.693147180559945309417;
  double r = 1. / 39916800;
  r = r * x + 1. / 3628800;
  r = r * x + 1. / 362880;
  r = r * x + 1. / 40320;
  r = r * x + 1. / 5040;
  r = r * x + 1. / 720;
  r = r * x + 1. / 120;
  r = r * x + 1. / 24;
  r = r * x + 1. / 6;
  r = r * x + 0.5;
  r = r * x + 1.;
  r = r * x + 1.;
  // (added to 2^52, the integer stands in the low bits)
  return (mass_t)(__double_as_longlong(__builtin_ldexp(r, (int)n + kFraction) + 4503599627370496.0) & 0xfffffffffffffll);
}

template <class T>
__device__ inline T wave_total(T x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  return x;
}
template <class T>
__device__ inline T wave_running(T x, int lane) {  // with the lane's own
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const T other = __shfl_up(x, d);
    if (lane >= d) x += other;
  }
  return x;
}

struct Row {
  uint32_t largest;  // key of the largest logit
  float top;         // its value
  double rate;       // log2 e / temperature
  __device__ double distance(float logit) const { return logit == top ? 0. : ((double)logit - (double)top) * rate; }
  __device__ mass_t weight(uint32_t key) const { return key == largest ? (mass_t)1 << kFraction : weight_of(distance(value_of(key))); }
};

// What stays of a row: keys above `key` and the first `ties` of those equal to it
struct Kept {
  uint32_t key;
  int ties;
};

struct Shared {
  uint32_t count[kBins];
  mass_t mass[kBins];
  mass_t parts[kWaves];
  mass_t above;
  mass_t other;
  uint32_t digit;
};

// The key in the falling order of those in `kept` behind which the running count or mass is `share` of the total or more (for counts: share is the count). In each
// pass the digit of 11 or 10 bits in whose bin that happens.
template <int TYPE, bool MASS>
__device__ Kept search(const void* logits, long long base, int vocabulary, const Row& row, const Kept& kept, double share, Shared& s) {
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  uint32_t prefix = 0;
  mass_t above = 0, target = 0;
  int shift = 21, bits = 11;
  const mass_t tied = kept.ties == INT_MAX ? 0 : (MASS ? row.weight(kept.key) : 1) * kept.ties;
  for (int level = 0; level < 3; ++level) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.mass[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < vocabulary; i += kThreads) {
      float x[1];
      load_values<TYPE, 1>(logits, base + i, x);
      const uint32_t key = key_of(x[0]);
      if (key <= kept.key && kept.ties != INT_MAX) continue;
      if (level && key >> (shift + bits) != prefix) continue;
      atomicAdd(&s.mass[key >> shift & ((1 << bits) - 1)], MASS ? row.weight(key) : 1);
    }
    __syncthreads();
    if (threadIdx.x == 0 && tied && (!level || kept.key >> (shift + bits) == prefix)) s.mass[kept.key >> shift & ((1 << bits) - 1)] += tied;
    __syncthreads();
    const mass_t first = s.mass[kBins - 1 - 2 * threadIdx.x], second = s.mass[kBins - 2 - 2 * threadIdx.x];
    const mass_t running = wave_running(first + second, lane);
    if (lane == 63) s.parts[wave] = running;
    __syncthreads();
    mass_t before = above, total = 0;
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) before += s.parts[w];
      total += s.parts[w];
    }
    if (level == 0) {
      target = MASS ? (mass_t)ceil(share * (double)total) : (mass_t)share;
      target = min(max(target, (mass_t)1), total);
    }
    before += running - first - second;
    if (before < target && before + first >= target) s.digit = kBins - 1 - 2 * threadIdx.x, s.above = before;
    before += first;
    if (before < target && before + second >= target) s.digit = kBins - 2 - 2 * threadIdx.x, s.above = before;
    __syncthreads();
    above = s.above;
    prefix = prefix << bits | s.digit;
    bits = level == 1 ? 10 : 11;
    shift = level == 0 ? 10 : 0;
    __syncthreads();
  }
  const mass_t each = MASS ? row.weight(prefix) : 1;
  return {prefix, (int)((target - above + each - 1) / each)};
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void sample_kernel(onebit_sampling a) {
  __shared__ Shared s;
  const int row_at = blockIdx.x, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const long long base = row_at * a.logits_stride;
  const float temperature = a.temperatures ? a.temperatures[row_at] : a.temperature;
  const float top_p = a.top_ps ? a.top_ps[row_at] : a.top_p, min_p = a.min_ps ? a.min_ps[row_at] : a.min_p;
  const int top_k = a.top_ks ? a.top_ks[row_at] : a.top_k;

  // the largest, of equals the lowest index; NaN
  mass_t best = 0;
  for (int i = threadIdx.x; i < a.vocabulary; i += kThreads) {
    float x[1];
    load_values<TYPE, 1>(a.logits, base + i, x);
    const mass_t own = x[0] != x[0] ? ~(mass_t)0 : (mass_t)key_of(x[0]) << 32 | (0xffffffffu - i);
    best = own > best ? own : best;
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const mass_t other = __shfl_xor(best, d);
    best = other > best ? other : best;
  }
  if (lane == 0) s.parts[wave] = best;
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) best = s.parts[w] > best ? s.parts[w] : best;
  __syncthreads();
  Row row;
  row.largest = (uint32_t)(best >> 32);
  if (best == ~(mass_t)0 || row.largest == kKeyOfMinusInfinity) {
    if (threadIdx.x == 0) a.tokens[row_at] = -1;
    return;
  }
  if (!(temperature > 0.f) || top_k == 1 || min_p > 1.f) {  // the first token alone
    if (threadIdx.x == 0) a.tokens[row_at] = 0xffffffffu - (uint32_t)best;
    return;
  }
  row.top = value_of(row.largest);
  row.rate = 1.44269504088896340736 / (double)temperature;
  const double least = min_p > 0.f ? log2((double)min_p) : -__builtin_inf();

  Kept kept = {0, INT_MAX};
  if (top_k > 0 && top_k < a.vocabulary) kept = search<TYPE, false>(a.logits, base, a.vocabulary, row, kept, top_k, s);
  if (top_p < 1.f) kept = search<TYPE, true>(a.logits, base, a.vocabulary, row, kept, fmaxf(top_p, 0.f), s);

  // masses of the wavefronts' own parts of the row, in the order of the indices
  const int part = (a.vocabulary + 64 * kWaves - 1) / (64 * kWaves) * 64, begin = min(wave * part, a.vocabulary), end = min(begin + part, a.vocabulary);
  auto stays = [&](float x) { return row.distance(x) >= least; };
  mass_t mass = 0;
  uint32_t ties = 0;
  for (int i = begin + lane; i < end; i += 64) {
    float x[1];
    load_values<TYPE, 1>(a.logits, base + i, x);
    const uint32_t key = key_of(x[0]);
    if (kept.ties != INT_MAX && key == kept.key) ++ties;
    else if (key >= kept.key && stays(x[0])) mass += row.weight(key);
  }
  ties = wave_total(ties);
  mass = wave_total(mass);
  if (lane == 0) s.parts[wave] = mass, s.count[wave] = ties;
  __syncthreads();
  const mass_t each = stays(value_of(kept.key)) ? row.weight(kept.key) : 0;
  mass_t before = 0, total = 0, own = 0;
  uint32_t ties_before = 0, own_ties_before = 0;
  for (int w = 0; w < kWaves; ++w) {
    const uint32_t left = (uint32_t)kept.ties > ties_before ? (uint32_t)kept.ties - ties_before : 0;
    const mass_t of_wave = s.parts[w] + each * min(left, s.count[w]);
    if (w == wave) before = total, own = of_wave, own_ties_before = ties_before;
    total += of_wave;
    ties_before += s.count[w];
  }
  const float u = a.uniform[row_at];
  const double at = u > 0.f ? (double)u * (double)total : 0.;
  const mass_t target = at < (double)total ? min((mass_t)at, total - 1) : total - 1;
  if (target < before || target >= before + own) return;
  mass_t running = before;
  for (int i = begin; i < end; i += 64) {
    float x[1] = {0.f};
    if (i + lane < end) load_values<TYPE, 1>(a.logits, base + i + lane, x);
    const uint32_t key = key_of(x[0]);
    const bool tie = i + lane < end && kept.ties != INT_MAX && key == kept.key;
    const mass_t tied = __ballot(tie);
    const uint32_t rank = own_ties_before + __popcll(tied & (((mass_t)1 << lane) - 1));
    mass_t w = 0;
    if (tie) w = rank < (uint32_t)kept.ties ? each : 0;
    else if (i + lane < end && key >= kept.key && stays(x[0])) w = row.weight(key);
    const mass_t sum = running + wave_running(w, lane);
    const mass_t over = __ballot(sum > target);
    if (over) {
      if (lane == 0) a.tokens[row_at] = i + __builtin_ctzll(over);
      return;
    }
    running = __shfl(sum, 63);
    own_ties_before += __popcll(tied);
  }
}

template <int TYPE>
hipError_t launch_as(const onebit_sampling& a, hipStream_t stream) {
  return launch_kernel(sample_kernel<TYPE>, dim3(a.rows), dim3(kThreads), 0, stream, a);
}

}  // namespace

hipError_t launch_sample(const onebit_sampling& a, hipStream_t stream) {
  if (a.logits_dtype == ONEBIT_DTYPE_F32) return launch_as<ONEBIT_DTYPE_F32>(a, stream);
  return a.logits_dtype == ONEBIT_DTYPE_F16 ? launch_as<ONEBIT_DTYPE_F16>(a, stream) : launch_as<ONEBIT_DTYPE_BF16>(a, stream);
}

}  // namespace onebit
