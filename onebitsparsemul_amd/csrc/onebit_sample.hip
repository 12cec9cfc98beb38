// Tokens from logits (onebit_head.h). Nothing is sorted: what the filters keep lies above a value, with those of the logits equal to it that have the lowest indices, so
// that a filter is a search for that value, a digit after the other in a histogram of counts or masses. Masses are integers (2^-42 of the largest
// weight): their sums do not depend on an order, and 2^-43 is the most a weight is off, so that which token a number falls on is what 64-bit sums give.
//
// A row is looked at once in full: the largest of each group of neighbouring logits stays. The k largest logits are not below the k-th largest of the groups' largest, and
// those that make up a share of the mass not below the value above which the groups' largest make it up alone; so that the filters
// see a list of few candidates, from the few groups that reach that value, in the order of their indices. Where a list would not hold them they go over the row's groups instead.
//
// Many rows are bound by the one pass over the logits (256 x 131072 fp32: 25 us, 5.3 TB/s), few by the second kernel's chain of steps over barriers, 8 to 10 us whatever the number of rows;
// 64 rows of 4096, in one kernel, 5.6. Rows with some hundred candidates take 6 to 10 us more, and one that keeps more than a list holds 86 to 207 of 131072 logits (256 such rows 123 to 271) and 35 to 74 of 32000, for the
// arithmetic of its weights in one workgroup.
#include "onebit_decoder_device.h"
#include "onebit_head_launch.h"

#include <algorithm>

namespace onebit {
namespace {

constexpr int kBins = 2048, kFraction = 42, kAll = INT_MAX;
constexpr float kFarthest = 50.f;
constexpr int kGroup = 16, kGroups = 8192;        // logits of a group, or that times a power of two; groups of a row
constexpr int kChunk = 4096, kChunkThreads = 256;  // logits of a workgroup of the first pass
typedef unsigned long long mass_t;

// Floats as integers of the same order; -0 as 0.
__device__ inline uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ inline float value_of(uint32_t key) { return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xffffffffu)); }
constexpr uint32_t kKeyOfNan = 0xffffffffu, kLeast = 0x00800000u, kNothing = 0;  // the key of the lowest finite logit; nothing: below all
__device__ inline uint32_t key_or_nan(float x) { return x != x ? kKeyOfNan : key_of(x); }

// 2^(x + 42) as an integer, x <= 0: 2^n r, r by the exponential series of the fraction of x, at most 1/2 of either sign: its twelve terms leave 2e-14 out.
__device__ __forceinline__ mass_t power_as_integer(double x) {
  if (!(x >= -kFraction - 1)) return 0;
  const double n = __builtin_rint(x), f = (x - n) * 0.693147180559945309417;
  double r = 1. / 39916800;
  r = r * f + 1. / 3628800;
  r = r * f + 1. / 362880;
  r = r * f + 1. / 40320;
  r = r * f + 1. / 5040;
  r = r * f + 1. / 720;
  r = r * f + 1. / 120;
  r = r * f + 1. / 24;
  r = r * f + 1. / 6;
  r = r * f + 0.5;
  r = r * f + 1.;
  r = r * f + 1.;
  // (added to 2^52, the integer stands in the low bits)
  return (mass_t)(__double_as_longlong(__builtin_ldexp(r, (int)n + kFraction) + 4503599627370496.0) & 0xfffffffffffffll);
}

// Weights beside the row's, or a part's, largest logit
struct Scale {
  uint32_t largest;  // its key
  float top;         // its value
  double rate;       // log2 e / temperature
  __device__ __forceinline__ Scale(uint32_t key, float temperature) : largest(key), top(value_of(key)), rate(1.44269504088896340736 / (double)temperature) {}
  __device__ __forceinline__ double distance(float logit) const { return logit == top ? 0. : ((double)logit - (double)top) * rate; }
  __device__ __forceinline__ mass_t weight(uint32_t key) const { return key == largest ? (mass_t)1 << kFraction : power_as_integer(distance(value_of(key))); }
};

struct Parameters {
  float temperature, top_p, min_p;
  int top_k;
  bool greedy, masses;  // the first token alone; all of the row's mass counts
  __device__ Parameters(const onebit_sampling& a, int row) {
    temperature = a.temperatures ? a.temperatures[row] : a.temperature;
    top_p = a.top_ps ? a.top_ps[row] : a.top_p;
    min_p = a.min_ps ? a.min_ps[row] : a.min_p;
    top_k = a.top_ks ? a.top_ks[row] : a.top_k;
    if (top_k <= 0 || top_k >= a.vocabulary) top_k = kAll;
    greedy = !(temperature > 0.f) || top_k == 1 || min_p > 1.f || top_p <= 0.f;
    masses = !greedy && top_k == kAll && (top_p < 1.f || !(min_p > 0.f));
  }
};

// Running sums over the lanes, with the lane's own: within rows of 16 by moves of 1, 2, 4 and 8 lanes, then the rows' last lanes to the rows behind.
template <int CTRL, int ROWS, class T>
__device__ inline T moved(T x) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, ROWS, 0xf, false));
  } else {
    const u2_t v = __builtin_bit_cast(u2_t, x);
    return __builtin_bit_cast(T, u2_t{(uint32_t)__builtin_amdgcn_update_dpp(0, (int)v.x, CTRL, ROWS, 0xf, false), (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v.y, CTRL, ROWS, 0xf, false)});
  }
}
template <class T>
__device__ inline T row_running(T x) {
  x += moved<0x111, 0xf>(x);
  x += moved<0x112, 0xf>(x);
  x += moved<0x114, 0xf>(x);
  return x + moved<0x118, 0xf>(x);
}
template <class T>
__device__ inline T wave_running(T x) {
  x = row_running(x);
  x += moved<0x142, 0xa>(x);
  return x + moved<0x143, 0xc>(x);
}
template <class T>
__device__ inline T of_lane(T x, int lane) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
  } else {
    const u2_t v = __builtin_bit_cast(u2_t, x);
    return __builtin_bit_cast(T, u2_t{(uint32_t)__builtin_amdgcn_readlane((int)v.x, lane), (uint32_t)__builtin_amdgcn_readlane((int)v.y, lane)});
  }
}
__device__ inline mass_t wave_most(mass_t x) {
  auto larger = [](mass_t a, mass_t b) { return a > b ? a : b; };
  x = larger(x, moved<0x111, 0xf>(x));
  x = larger(x, moved<0x112, 0xf>(x));
  x = larger(x, moved<0x114, 0xf>(x));
  x = larger(x, moved<0x118, 0xf>(x));
  x = larger(x, moved<0x142, 0xa>(x));
  return of_lane(larger(x, moved<0x143, 0xc>(x)), 63);
}

// f of each of four, or eight, keys: once in the code, which is fetched anew by every launch's workgroups and costs them more than the moves
template <class F>
__device__ __forceinline__ void each_of(u4_t four, F f) {
#pragma unroll 1
  for (int e = 0; e < 4; ++e) {
    f(four.x);
    four = u4_t{four.y, four.z, four.w, four.x};
  }
}
template <class F>
__device__ __forceinline__ void each_of(u4_t one, u4_t other, F f) {
#pragma unroll 1
  for (int e = 0; e < 8; ++e) {
    f(one.x);
    const uint32_t first = one.x;
    one = u4_t{one.y, one.z, one.w, other.x};
    other = u4_t{other.y, other.z, other.w, first};
  }
}

// What stays of a row: keys above `key` and the first `ties` of those equal to it
struct Kept {
  uint32_t key;
  int ties;
};

// Candidates of a list: what LDS holds. (A compute unit has one workgroup of 1024 threads with lists of 4096, too.)
template <int THREADS>
struct Shared {
  static constexpr int kListed = THREADS == 1024 ? 14336 : 4096;
  mass_t bins[kBins];
  __attribute__((aligned(16))) uint32_t keys[kListed + 4];
  uint32_t indices[kListed + 4];  // candidates in the order of their indices
  uint32_t reaching[kGroups / 2];            // groups that reach the candidates' value, 16 bits each
  mass_t parts[2][THREADS / 64];
  mass_t above, few_amounts[64];
  uint32_t bin, few, few_keys[64];  // a bin's items
};

// A workgroup of THREADS on a row
template <int THREADS>
struct Block {
  static constexpr int kWaves = THREADS / 64;  // at most 16: the lanes of a row
  static constexpr int kListed = Shared<THREADS>::kListed;
  Shared<THREADS>& s;
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  int turn = 0;  // which of the parts is next, so that one barrier does
  __device__ Block(Shared<THREADS>& shared) : s(shared) {}

  // Each wavefront's part, over a barrier: lane w has that of wavefront w
  template <class T>
  __device__ T part_of_lane(T own) {
    T* const parts = (T*)s.parts[turn ^= 1];
    if (lane == 0) parts[wave] = own;
    __syncthreads();
    return parts[lane % kWaves];
  }
  __device__ mass_t most(mass_t x) { return wave_most(part_of_lane(wave_most(x))); }
  // sum of the threads in front, and of all
  template <class T>
  __device__ T before(T x, T& total) {
    const T running = wave_running(x), parts = row_running(part_of_lane(of_lane(running, 63)));
    total = of_lane(parts, kWaves - 1);
    return running - x + (wave ? of_lane(parts, wave - 1) : 0);
  }

  // The bin in which the running sum over the bins, `above` in front of them, comes to `target`, into s.bin, and the sum in front of it into s.above, for after the next barrier
  __device__ __forceinline__ bool locate(mass_t target, mass_t above) {
    constexpr int kEach = kBins / THREADS;
    mass_t own[kEach], sum = 0, total;
#pragma unroll
    for (int i = 0; i < kEach; ++i) sum += own[i] = s.bins[threadIdx.x * kEach + i];
    mass_t front = above + before(sum, total);
    if (above + total < target) return false;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (front < target && front + own[i] >= target) s.bin = threadIdx.x * kEach + i, s.above = front;
      front += own[i];
    }
    return true;
  }

  // The key, from `high` down to `low`, with which the running sum of the items' amounts comes to `target` or more, the sum in front of it, and whether it comes to it. each(f) calls
  // f(key) for the thread's items; of key `extra` there is extra_amount once. In each round the bin of 2^shift keys in which that happens; LISTED: its items, where
  // they are at most 64, are compared with each other (two rounds less: top_k 500 and top_p 0.9 of 719 candidates 6.1 us for 9.5).
  template <bool LISTED, class Each, class Amount>
  __device__ __forceinline__ bool search(uint32_t high, uint32_t low, mass_t target, Each each, Amount amount, uint32_t extra, mass_t extra_amount, uint32_t& key, mass_t& in_front) {
    mass_t above = 0;
    for (;;) {
      const int shift = max(0, 32 - __clz((int)(high - low)) - 11);
      for (int i = threadIdx.x; i < kBins; i += THREADS) s.bins[i] = 0;
      __syncthreads();
      each([&](uint32_t own) {
        if (own <= high && own >= low) atomicAdd(&s.bins[(high - own) >> shift], amount(own));
      });
      if (threadIdx.x == 0 && extra_amount && extra <= high && extra >= low) atomicAdd(&s.bins[(high - extra) >> shift], extra_amount);
      __syncthreads();
      if (!locate(target, above)) return false;  // (in the first round, and for all threads)
      if (LISTED && threadIdx.x == 0) s.few = 0;
      __syncthreads();
      above = s.above;
      high -= s.bin << shift;
      low = max(low, high - ((1u << shift) - 1));
      if (shift == 0) break;
      if (LISTED) {
        auto take = [&](uint32_t own, mass_t amount) {
          if (const uint32_t at = atomicAdd(&s.few, 1u); at < 64) s.few_keys[at] = own, s.few_amounts[at] = amount;
        };
        each([&](uint32_t own) {
          if (own <= high && own >= low) take(own, amount(own));
        });
        if (threadIdx.x == 0 && extra_amount && extra <= high && extra >= low) take(extra, extra_amount);
        __syncthreads();
        const int few = __builtin_amdgcn_readfirstlane((int)s.few);
        if (few <= 64) {
          const uint32_t own_key = s.few_keys[lane];
          mass_t larger = above, with = above;
          for (int j = 0; j < few; ++j) {
            const uint32_t other = s.few_keys[j];
            const mass_t amount = s.few_amounts[j];
            larger += other > own_key ? amount : 0;
            with += other >= own_key ? amount : 0;
          }
          const int here = __builtin_ctzll(__ballot(lane < few && larger < target && with >= target));
          high = (uint32_t)of_lane((int)own_key, here), above = of_lane(larger, here);
          break;
        }
      }
    }
    key = high;
    in_front = above;
    return true;
  }

  // The same of items that take long to look at: once for bins that are as wide as each other in logits, once for a list of that bin's, in which the rest is found. (A row of 131072 of
  // which top_p keeps most: 200 us, with rounds over all of them 252.)
  template <class Each, class Amount>
  __device__ __forceinline__ bool search_many(uint32_t high, uint32_t low, mass_t target, Each each, Amount amount, uint32_t extra, mass_t extra_amount, uint32_t& key, mass_t& in_front) {
    const float top = value_of(high), width = (kBins - 1) / (top - value_of(low));
    auto place = [&](uint32_t own) { return (uint32_t)fminf((top - value_of(own)) * width, kBins - 1.f); };  // (NaN, of infinities: the last)
    for (int i = threadIdx.x; i < kBins; i += THREADS) s.bins[i] = 0;
    __syncthreads();
    each([&](uint32_t own) {
      if (own <= high && own >= low) atomicAdd(&s.bins[place(own)], amount(own));
    });
    if (threadIdx.x == 0 && extra_amount && extra <= high && extra >= low) atomicAdd(&s.bins[place(extra)], extra_amount);
    __syncthreads();
    if (!locate(target, 0)) return false;
    if (threadIdx.x == 0) s.few = 0;
    __syncthreads();
    const uint32_t bin = s.bin;
    const mass_t above = s.above;
    each([&](uint32_t own) {
      if (own <= high && own >= low && place(own) == bin)
        if (const uint32_t at = atomicAdd(&s.few, 1u); at < kListed) s.keys[at] = own;
    });
    __syncthreads();
    const int count = (int)s.few;
    if (count > kListed) return search<false>(high, low, target, each, amount, extra, extra_amount, key, in_front);
    auto each_listed = [&](auto f) {
      for (int i = threadIdx.x; i < count; i += THREADS) f(s.keys[i]);
    };
    if (extra_amount && (extra > high || extra < low || place(extra) != bin)) extra_amount = 0;
    search<true>(high, low, target - above, each_listed, amount, extra, extra_amount, key, in_front);
    in_front += above;
    return true;
  }
  template <bool LISTED, class Each, class Amount>
  __device__ __forceinline__ bool search_any(uint32_t high, uint32_t low, mass_t target, Each each, Amount amount, uint32_t extra, mass_t extra_amount, uint32_t& key, mass_t& in_front) {
    if constexpr (LISTED) return search<true>(high, low, target, each, amount, extra, extra_amount, key, in_front);
    else return search_many(high, low, target, each, amount, extra, extra_amount, key, in_front);
  }
};

// The filters by rank and by share. each(f) calls f(key) for the thread's items, all of them from key `low` on, in any order; mass: the row's, where it counts.
template <bool LISTED, int THREADS, class Each>
__device__ __forceinline__ Kept filtered(Block<THREADS>& block, const Scale& scale, const Parameters& p, uint32_t low, double mass, Each each) {
  Kept kept = {kNothing, kAll};
  uint32_t key;
  mass_t in_front;
  if (p.top_k != kAll && block.template search_any<LISTED>(scale.largest, low, p.top_k, each, [](uint32_t) { return (mass_t)1; }, 0, 0, key, in_front)) kept = {key, p.top_k - (int)in_front};
  if (p.top_p < 1.f) {
    const mass_t tied = kept.ties == kAll ? 0 : scale.weight(kept.key) * kept.ties;
    auto above = [&](auto f) {
      each([&](uint32_t own) {
        if (own > kept.key || kept.ties == kAll) f(own);
      });
    };
    if (p.top_k != kAll) {  // of those that top_k left
      mass_t own_mass = threadIdx.x == 0 ? tied : 0, total;
      above([&](uint32_t own) { own_mass += own >= low ? scale.weight(own) : 0; });
      block.before(own_mass, total);
      mass = (double)total;
    }
    // (where rounding leaves the running sum below: all stay)
    const mass_t target = max((mass_t)ceil((double)p.top_p * mass), (mass_t)1);
    if (block.template search_any<LISTED>(scale.largest, max(low, kept.key), target, above, [&](uint32_t own) { return scale.weight(own); }, kept.key, tied, key, in_front)) {
      const mass_t one = scale.weight(key);
      kept = {key, (int)((target - in_front + one - 1) / one)};
    }
  }
  return kept;
}

// The weight of an item in the last sum: 0 where min_p leaves it out
struct Last {
  const Scale& scale;
  double least;
  __device__ __forceinline__ Last(const Scale& s, const Parameters& p) : scale(s), least(p.min_p > 0.f ? log2((double)p.min_p) : -__builtin_inf()) {}
  __device__ __forceinline__ mass_t weight(uint32_t key) const { return scale.distance(value_of(key)) >= least ? scale.weight(key) : 0; }
};
__device__ inline mass_t target_of(float uniform, double total, mass_t whole) {
  const double at = uniform > 0.f ? (double)uniform * total : 0.;
  return at < total ? min((mass_t)at, whole - 1) : whole - 1;
}

// Items in fours: keys(i) gives those of items 4 i ... 4 i + 3, i < count, in the order of their indices, index(item) an item's. Of those that `kept` leaves, the first at which
// the running mass exceeds `at`, or uniform times the total where `at` is negative. Each wavefront sums a stretch, 64 fours at a time; the stretch in which it happens is
// shared out again until one wavefront walks through it.
template <int THREADS, class Keys, class Index>
__device__ __forceinline__ void choose(Block<THREADS>& block, const Last& last, const Kept& kept, float uniform, double at, int count, Keys keys, Index index, long long* token) {
  const bool bounded = kept.ties != kAll;
  const mass_t each = bounded ? last.weight(kept.key) : 0;
  const int lane = block.lane;
  int first = 0;
  mass_t front = 0, left = bounded ? (mass_t)kept.ties : 0, target = 0;  // in front of the items, ties that they may keep
  for (bool whole = true;; whole = false) {
    const int stretch = (count + THREADS - 1) / THREADS * 64, begin = first + min(block.wave * stretch, count), end = min(begin + stretch, first + count);
    mass_t ties = 0, mass = 0, total;
    constexpr u4_t kNone = {kNothing, kNothing, kNothing, kNothing};
    for (int i = begin + lane; i < end; i += 128) {
      const u4_t one = keys(i), other = i + 64 < end ? keys(i + 64) : kNone;
      each_of(one, other, [&](uint32_t key) {
        const bool tie = bounded && key == kept.key;
        ties += tie;
        mass += key >= kept.key && key >= kLeast && !tie ? last.weight(key) : 0;
      });
    }
    mass_t in_front = 0;  // ties in front of the wavefront's
    if (each) {
      mass_t ignored;
      in_front = of_lane(block.before(ties, ignored), 0);
      const mass_t of_wave = of_lane(wave_running(ties), 63), may = left > in_front ? left - in_front : 0;
      if (lane == 0) mass += min(may, of_wave) * each;
    }
    const mass_t running = front + of_lane(block.before(mass, total), 0), of_wave = of_lane(wave_running(mass), 63);
    if (whole) target = at < 0. ? target_of(uniform, (double)total, total) : min((mass_t)at, total - 1);
    const bool here = running <= target && running + of_wave > target;
    left = left > in_front ? left - in_front : 0;
    if (stretch <= 64 * 4) {
      if (!here) return;
      first = begin, count = end - begin, front = running;
      break;
    }
    if (here && lane == 0) block.s.bins[0] = (mass_t)begin, block.s.bins[1] = (mass_t)end, block.s.bins[2] = running, block.s.bins[3] = left;
    __syncthreads();
    first = (int)block.s.bins[0], count = (int)block.s.bins[1] - first, front = block.s.bins[2], left = block.s.bins[3];
    __syncthreads();
  }
  for (int i = first; i < first + count; i += 64) {
    u4_t four = {kNothing, kNothing, kNothing, kNothing};
    if (i + lane < first + count) four = keys(i + lane);
    int ties = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) ties += bounded && four[e] == kept.key;
    const int ties_running = wave_running(ties);
    mass_t may = (mass_t)(ties_running - ties);
    may = left > may ? left - may : 0;
    mass_t own = 0;
    auto weigh = [&](uint32_t key, mass_t& may) -> mass_t {
      if (bounded && key == kept.key) {
        const mass_t w = may ? each : 0;
        may -= may ? 1 : 0;
        return w;
      }
      return key >= kept.key && key >= kLeast ? last.weight(key) : 0;
    };
    const mass_t may_at_first = may;
    each_of(four, [&](uint32_t key) { own += weigh(key, may); });
    const mass_t running = wave_running(own), over = __ballot(front + running > target);
    if (over) {
      if (lane == __builtin_ctzll(over)) {
        mass_t sum = front + running - own;
        int found = 0;
        may = may_at_first;
        each_of(four, [&](uint32_t key) { found += (sum += weigh(key, may)) <= target; });
        *token = index(4 * (i + lane) + found);
      }
      return;
    }
    front += of_lane(running, 63);
    const mass_t all = (mass_t)of_lane(ties_running, 63);
    left = left > all ? left - all : 0;
  }
}

// Few candidates: each is compared with each other, wavefronts taking every so manieth of them: how many are in front of it, and their mass
// (with 256 threads 100 take 13.7 us in this way and 12.5 in the other, with 512 150 11.5 and 12.0, with 1024 200 15.6 and 16.2)
template <int THREADS>
constexpr int kPaired = 64 + THREADS / 8;
template <int THREADS>
__device__ __forceinline__ void choose_of_few(Block<THREADS>& block, const Scale& scale, const Last& last, const Parameters& p, double mass, float uniform, int count, long long* token) {
  Shared<THREADS>& s = block.s;
  constexpr int kMost = kPaired<THREADS>;
  mass_t *const weights = s.bins, *const fronts = s.bins + kMost, *const ranks = s.bins + 2 * kMost;
  const int own = threadIdx.x;
  if (own < count) weights[own] = scale.weight(s.keys[own]), fronts[own] = ranks[own] = 0;
  __syncthreads();
  for (int i = block.lane; i < count; i += 64) {
    const uint32_t key = s.keys[i];
    mass_t front = 0;
    int rank = 0;
#pragma unroll 4
    for (int j = block.wave; j < count; j += THREADS / 64) {
      const uint32_t other = s.keys[j];
      const bool better = other > key || (other == key && j < i);
      rank += better;
      front += better ? weights[j] : 0;
    }
    if (rank) atomicAdd(&ranks[i], (mass_t)rank), atomicAdd(&fronts[i], front);
  }
  __syncthreads();
  const bool there = own < count;
  bool stays = there && ranks[own] < (mass_t)p.top_k;
  if (p.top_p < 1.f) {
    if (p.top_k != kAll) {
      mass_t total;
      block.before(stays ? weights[own] : 0, total);
      mass = (double)total;
    }
    stays = stays && fronts[own] < max((mass_t)ceil((double)p.top_p * mass), (mass_t)1);
  }
  const mass_t w = stays ? last.weight(s.keys[own]) : 0;
  mass_t total;
  const mass_t front = block.before(w, total), target = target_of(uniform, (double)total, total);
  if (front <= target && front + w > target) *token = s.indices[own];
}

// The row's groups of `group` logits: the thread's are kCount from number `first` on, their largest keys as given; four_at(i): the keys of logits i ... i + 3, i a multiple of four.
template <int THREADS, int kCount, class Key>
__device__ __forceinline__ void sample_row(Block<THREADS>& block, const uint32_t (&most)[kCount], int first, int group, Key four_at, const onebit_sampling& a, int row, const Scale& scale,
                           const Parameters& p, double mass) {
  constexpr int kListed = Shared<THREADS>::kListed;
  Shared<THREADS>& s = block.s;
  // A value that all candidates reach. Weights 2^-50 of the largest are 0: no such logit matters, whatever its rank.
  const float steep = (float)scale.rate;
  float distance[kCount], reach = kFarthest;
#pragma unroll
  for (int i = 0; i < kCount; ++i) distance[i] = most[i] >= kLeast ? most[i] == scale.largest ? 0.f : (scale.top - value_of(most[i])) * steep : INFINITY;
  if (p.top_k != kAll || p.top_p < 1.f) {
    // The groups' largest within `reach` are top_k, or have top_p of the mass: from a histogram of their distances, 256 bins for each doubling of an eighth and the distance. First with the
    // threads' largest alone; where they do not come to it, or would be most of them, with all (top_k 1000 and top_p 0.9 of 131072, 16 rows: 24.6 us, by the threads' largest 153). Masses in 2^-31 of the row's, cut off, and with some room.
    const bool by_rank = p.top_k != kAll;
    const float unit = by_rank ? 1.f : (float)(0x1p73 / mass);
    const mass_t target = by_rank ? (mass_t)p.top_k : (mass_t)((double)p.top_p * 0x1p31 * (1. + 0x1p-10)) + 1;
    uint32_t* const bins = (uint32_t*)s.bins;
    constexpr uint32_t kEighth = 0x3e000000u, kEdges = ((0x42488000u - kEighth) >> 15) + 1;  // (50 and an eighth)
    constexpr int kEach = (kEdges + THREADS - 1) / THREADS;
    static_assert(sizeof(s.bins) >= kEach * THREADS * sizeof(uint32_t), "");
    auto add = [&](float d) {
      if (d <= kFarthest) atomicAdd(&bins[(__float_as_uint(d + 0.125f) - kEighth) >> 15], by_rank ? 1u : (uint32_t)(__builtin_amdgcn_exp2f(-d) * unit));
    };
    float nearest = distance[0];
#pragma unroll
    for (int i = 1; i < kCount; ++i) nearest = fminf(nearest, distance[i]);
#pragma unroll 1
    for (int pass = kCount > 1 && by_rank && p.top_k > THREADS / 2; pass < (kCount > 1 ? 2 : 1); ++pass) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) bins[threadIdx.x + i * THREADS] = 0;
      __syncthreads();
      if (pass == 0) {
        add(nearest);
      } else {
#pragma unroll
        for (int i = 0; i < kCount; ++i) add(distance[i]);
      }
      __syncthreads();
      uint32_t own[kEach], sum = 0, total;
#pragma unroll
      for (int i = 0; i < kEach; ++i) sum += own[i] = bins[threadIdx.x * kEach + i];
      uint32_t front = block.before(sum, total);
      if (total < target) continue;  // (for all threads; the bins have been read)
      if (front < target && front + sum >= target) {
        uint32_t bin = threadIdx.x * kEach;
#pragma unroll
        for (int i = 0; i < kEach - 1; ++i)
          if ((front += own[i]) < target) ++bin;
        s.bin = bin;
      }
      __syncthreads();
      reach = __uint_as_float(((s.bin + 1) << 15) + kEighth) - 0.125f;
      break;
    }
  }
  // Nor does top_p need what lies so far that all of the vocabulary there would have less than the mass that it leaves out (by a factor of 2^-2^-9: of 2^-10 of the mass and more that is above
  // the logarithm's error and all weights' roundings, 2^-23 of the largest). Rows whose mass is spread over groups: 32000 under top_p 0.95 39 us, listed whole or by groups 71.
  if (p.top_k == kAll && p.top_p < 1.f - 0x1p-10f) reach = fminf(reach, __builtin_amdgcn_logf((float)(a.vocabulary / ((1. - (double)p.top_p) * mass * 0x1p-42))) + 0x1p-9f);
  // (a step further than fp32 rounds)
  const double farthest = (double)scale.top - ((double)reach * (1. + 0x1p-20) + 0x1p-20) / scale.rate;
  const float edge = (float)(farthest - fabs(farthest) * 0x1p-22);
  uint32_t low = edge == edge ? max(kLeast, key_of(edge)) : scale.largest;  // (NaN: +inf among the logits, and only such)
  mass_t total;
  const Last last(scale, p);
  const float uniform = a.uniform[row];
  long long* const token = a.tokens + row;
  // min_p comes behind the others: top_p's mass counts what it leaves out.
  if (p.min_p > 0.f && p.top_p >= 1.f) {
    const double least = (double)scale.top + last.least / scale.rate;
    const float least_edge = (float)(least - fabs(least) * 0x1p-22);
    if (least_edge == least_edge) low = max(low, key_of(least_edge));
  }
  // the groups that reach it, in order
  int own_groups = 0, reaching_groups;
#pragma unroll
  for (int i = 0; i < kCount; ++i) own_groups += most[i] >= low;
  int at = block.before(own_groups, reaching_groups);
  uint16_t* const reaching = (uint16_t*)s.reaching;
#pragma unroll
  for (int i = 0; i < kCount; ++i)
    if (most[i] >= low) reaching[at++] = (uint16_t)(first + i);
  const int fours = reaching_groups * group / 4, shift = __builtin_ctz(group) - 2;  // (at most the vocabulary, rounded up)
  __syncthreads();
  auto index_of_four = [&](int i) { return (int)reaching[i >> shift] * group + (i & (group / 4 - 1)) * 4; };
  auto four = [&](int i) { return four_at(index_of_four(i)); };
  // their logits that reach it, listed in order where they are few
  int listed = 0;
  constexpr int kBatch = 2;
  for (int i = 0; i < fours && listed <= kListed; i += kBatch * THREADS) {
    u4_t one[kBatch];
    int own[kBatch], in_front[kBatch], all[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int at = i + j * THREADS + threadIdx.x;
      one[j] = at < fours ? four(at) : u4_t{kNothing, kNothing, kNothing, kNothing};
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      own[j] = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) own[j] += one[j][e] >= low;
    }
    // (both at once, 16 bits each)
    const int both = block.before(own[0] | own[1] << 16, all[0]);
    in_front[0] = both & 0xffff, in_front[1] = both >> 16, all[1] = all[0] >> 16, all[0] &= 0xffff;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      int to = listed + in_front[j];
      if (own[j]) {
        const int index = index_of_four(i + j * THREADS + threadIdx.x);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (one[j][e] >= low) {
            if (to < kListed) s.keys[to] = one[j][e], s.indices[to] = index + e;
            ++to;
          }
      }
      listed += all[j];
    }
  }
  if (threadIdx.x < 4 && listed <= kListed) s.keys[listed + threadIdx.x] = kNothing;
  __syncthreads();
  if (listed <= kPaired<THREADS>) {
    choose_of_few(block, scale, last, p, mass, uniform, listed, token);
  } else if (listed <= kListed) {
    const Kept kept = filtered<true>(block, scale, p, low, mass, [&](auto f) {
      for (int i = threadIdx.x; i < listed; i += THREADS) f(s.keys[i]);
    });
    choose(block, last, kept, uniform, -1., (listed + 3) / 4, [&](int i) { return *(const u4_t*)(s.keys + 4 * i); }, [&](int i) { return (long long)s.indices[i]; }, token);
  } else {
    auto reached = [&](int i) {
      u4_t one = four(i);
#pragma unroll
      for (int e = 0; e < 4; ++e) one[e] = one[e] >= low ? one[e] : kNothing;
      return one;
    };
    const Kept kept = filtered<false>(block, scale, p, low, mass, [&](auto f) {
      for (int i = threadIdx.x; i < fours; i += 2 * THREADS) {
        const u4_t one = reached(i), other = i + THREADS < fours ? reached(i + THREADS) : u4_t{kNothing, kNothing, kNothing, kNothing};
        each_of(one, other, f);
      }
    });
    choose(block, last, kept, uniform, -1., fours, reached, [&](int i) { return (long long)index_of_four(i / 4) + i % 4; }, token);
  }
}

// N consecutive logits from `at` on as keys, nothing beyond the row's end
template <int TYPE, int N>
__device__ inline void load_keys(const void* logits, long long base, int at, int vocabulary, uint32_t (&keys)[N]) {
  typedef typename Stored<TYPE>::type T;
  constexpr int kOf16 = N < 16 / (int)sizeof(T) ? N : 16 / (int)sizeof(T);
  typedef T vector __attribute__((ext_vector_type(kOf16), aligned(sizeof(T))));  // (16 bytes from any address)
  const T* const from = (const T*)logits + base + at;
  if (at + N <= vocabulary) {
    vector v[N / kOf16];
#pragma unroll
    for (int i = 0; i < N / kOf16; ++i) v[i] = ((const vector*)from)[i];
#pragma unroll
    for (int i = 0; i < N; ++i) keys[i] = key_or_nan((float)v[i / kOf16][i % kOf16]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) keys[i] = at + i < vocabulary ? key_or_nan((float)from[i]) : kNothing;
  }
}
template <int N>
__device__ inline uint32_t most_of(const uint32_t (&keys)[N]) {
  uint32_t most = keys[0];
#pragma unroll
  for (int i = 1; i < N; ++i) most = max(most, keys[i]);
  return most;
}
// The largest with the lowest index of equals
template <int N>
__device__ inline mass_t first_most(const uint32_t (&keys)[N], uint32_t most, int at) {
  int first = N - 1;
#pragma unroll
  for (int i = N - 2; i >= 0; --i)
    if (keys[i] == most) first = i;
  return (mass_t)most << 32 | (0xffffffffu - (uint32_t)(at + first));
}
// The token where it follows from the largest alone
__device__ inline bool settled(mass_t best, const Parameters& p, long long* token) {
  const uint32_t key = (uint32_t)(best >> 32);
  const bool none = key == kKeyOfNan || key < kLeast;
  if (!none && !p.greedy) return false;
  if (threadIdx.x == 0) *token = none ? -1 : (long long)(0xffffffffu - (uint32_t)best);
  return true;
}

// A row in one workgroup's LDS
template <int TYPE, int THREADS, int MOST>
__global__ __launch_bounds__(THREADS) void sample_short_kernel(onebit_sampling a) {
  __shared__ Shared<THREADS> s;
  __shared__ __attribute__((aligned(16))) uint32_t row_keys[MOST];
  Block<THREADS> block(s);
  const int row = blockIdx.x;
  const Parameters p(a, row);
  constexpr int kCount = MOST / kGroup / THREADS;
  uint32_t most[kCount];
  mass_t best = 0;
#pragma unroll
  for (int g = 0; g < kCount; ++g) {
    const int at = (threadIdx.x * kCount + g) * kGroup;
    uint32_t keys[kGroup];
    load_keys<TYPE, kGroup>(a.logits, row * a.logits_stride, at, a.vocabulary, keys);
#pragma unroll
    for (int i = 0; i < kGroup; i += 4) *(u4_t*)(row_keys + at + i) = u4_t{keys[i], keys[i + 1], keys[i + 2], keys[i + 3]};
    most[g] = most_of(keys);
    const mass_t own = first_most(keys, most[g], at);
    best = own > best ? own : best;
  }
  best = block.most(best);  // (with a barrier: the keys are there)
  if (settled(best, p, a.tokens + row)) return;
  const Scale scale((uint32_t)(best >> 32), p.temperature);
  auto four_at = [&](int i) { return *(const u4_t*)(row_keys + i); };
  double mass = 0.;
  if (p.masses) {
    auto four_at_place = [&](int i) { return four_at(4 * i); };
    if (p.top_p >= 1.f) {  // no filter
      choose(block, Last(scale, p), {kNothing, kAll}, a.uniform[row], -1., (a.vocabulary + 3) / 4, four_at_place, [](int i) { return (long long)i; }, a.tokens + row);
      return;
    }
    mass_t own = 0, total;
    for (int i = threadIdx.x; i < a.vocabulary; i += THREADS) own += row_keys[i] >= kLeast ? scale.weight(row_keys[i]) : 0;
    block.before(own, total);
    mass = (double)total;
  }
  sample_row(block, most, threadIdx.x * kCount, kGroup, four_at, a, row, scale, p, mass);
}

// Long rows, first pass: a chunk's largest, its mass beside that where masses count, and its groups' largest
struct Chunks {
  mass_t *best, *mass;   // rows x chunks
  uint32_t* largest;     // rows x groups
  int chunks, groups;    // of a row
  int group;             // logits of a group
};
template <int TYPE>
__global__ __launch_bounds__(kChunkThreads) void chunk_kernel(onebit_sampling a, Chunks c) {
  __shared__ mass_t parts[2][kChunkThreads / 64];
  const int chunk = blockIdx.x, row = blockIdx.y, at = chunk * kChunk + threadIdx.x * kGroup, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const Parameters p(a, row);
  uint32_t keys[kGroup];
  load_keys<TYPE, kGroup>(a.logits, row * a.logits_stride, at, a.vocabulary, keys);
  const uint32_t most = most_of(keys);
  uint32_t of_group = most;
  for (int d = 1; d < c.group / kGroup; d <<= 1) of_group = max(of_group, (uint32_t)__shfl_xor((int)of_group, d));
  const int group = at / c.group;
  if (at % c.group == 0 && group < c.groups) c.largest[(long long)row * c.groups + group] = of_group;
  mass_t best = wave_most(first_most(keys, most, at));
  if (lane == 0) parts[0][wave] = best;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kChunkThreads / 64; ++w) best = parts[0][w] > best ? parts[0][w] : best;
  const uint32_t key = (uint32_t)(best >> 32);
  mass_t mass = 0;
  if (p.masses && key >= kLeast && key != kKeyOfNan) {
    const Scale scale(key, p.temperature);
#pragma unroll
    for (int i = 0; i < kGroup; i += 8)
      each_of(u4_t{keys[i], keys[i + 1], keys[i + 2], keys[i + 3]}, u4_t{keys[i + 4], keys[i + 5], keys[i + 6], keys[i + 7]},
              [&](uint32_t key) { mass += key >= kLeast ? scale.weight(key) : 0; });
    mass = of_lane(wave_running(mass), 63);
    if (lane == 0) parts[1][wave] = mass;
    __syncthreads();
    mass = 0;
#pragma unroll
    for (int w = 0; w < kChunkThreads / 64; ++w) mass += parts[1][w];
  }
  if (threadIdx.x == 0) {
    c.best[(long long)row * c.chunks + chunk] = best;
    c.mass[(long long)row * c.chunks + chunk] = mass;
  }
}

constexpr int kLongThreads = 1024;
template <int TYPE>
__global__ __launch_bounds__(kLongThreads) void sample_long_kernel(onebit_sampling a, Chunks c) {
  __shared__ Shared<kLongThreads> s;
  Block<kLongThreads> block(s);
  const int row = blockIdx.x;
  const Parameters p(a, row);
  const mass_t own_best = (int)threadIdx.x < c.chunks ? c.best[(long long)row * c.chunks + threadIdx.x] : 0;
  const mass_t best = block.most(own_best);
  if (settled(best, p, a.tokens + row)) return;
  const Scale scale((uint32_t)(best >> 32), p.temperature);
  auto four_at = [&](int i) {
    uint32_t keys[4];
    load_keys<TYPE, 4>(a.logits, row * a.logits_stride, i, a.vocabulary, keys);
    return u4_t{keys[0], keys[1], keys[2], keys[3]};
  };
  double mass = 0.;
  if (p.masses) {
    // The chunks' masses in the row's unit, in their order: 64 bits of a float, rounded alike each time
    // (one whose largest's weight rounds to 0 beside the row's has none)
    double own = 0.;
    const uint32_t own_key = (uint32_t)(own_best >> 32);
    if (own_key >= kLeast && scale.weight(own_key) != 0) own = (double)c.mass[(long long)row * c.chunks + threadIdx.x] * exp2(scale.distance(value_of(own_key)));
    // (at most 256 chunks: four wavefronts)
    double* const sums = (double*)s.bins;
    const double running = wave_running(own);
    if (block.lane == 63) sums[block.wave] = running;
    __syncthreads();
    double front = running - own;
    for (int w = 0; w < 4; ++w) {
      if (w < block.wave) front += sums[w];
      mass += sums[w];
    }
    if (p.top_p >= 1.f) {  // no filter: the chunk, then the token in it
      const float uniform = a.uniform[row];
      const double at = uniform > 0.f ? (uniform < 1.f ? (double)uniform * mass : INFINITY) : 0.;  // (NaN: 0)
      const mass_t beyond = front + own > at && own > 0. ? 1 : 0, any = own > 0. ? 1 : 0;
      // the first chunk beyond, or the last one with a mass
      const mass_t found = block.most(beyond ? (mass_t)1 << 40 | (mass_t)(kLongThreads - threadIdx.x) : any ? (mass_t)threadIdx.x + 1 : 0);
      const bool over = found >> 40;
      const int chunk = over ? kLongThreads - (int)(found & 0xffffffff) : (int)found - 1;
      // (of chunks whose sums are rounded, one may begin behind the number that the one in front of it does not come to: its first token)
      if ((int)threadIdx.x == chunk) ((double*)s.bins)[16] = over ? fmax(at - front, 0.) : 0x1p62;
      __syncthreads();
      const double rest = ((double*)s.bins)[16];
      const int begin = chunk * kChunk, count = min(kChunk, a.vocabulary - begin);
      choose(block, Last(scale, p), {kNothing, kAll}, uniform, rest, (count + 3) / 4, [&](int i) { return four_at(begin + 4 * i); }, [&](int i) { return (long long)(begin + i); }, a.tokens + row);
      return;
    }
    __syncthreads();  // the sums' readers are through
  }
  constexpr int kCount = kGroups / kLongThreads;
  const int share = (c.groups + kLongThreads - 1) / kLongThreads, first = threadIdx.x * share;  // at most kCount
  uint32_t most[kCount];
#pragma unroll
  for (int i = 0; i < kCount; ++i) most[i] = kNothing;
  const uint32_t* const largest = c.largest + (long long)row * c.groups;
  if (share == kCount && first + kCount <= c.groups) {
    typedef uint32_t vector __attribute__((ext_vector_type(4), aligned(4)));  // (16 bytes from any address)
    static_assert(kCount % 4 == 0, "");
#pragma unroll
    for (int i = 0; i < kCount; i += 4) {
      const vector v = *(const vector*)(largest + first + i);
      most[i] = v.x, most[i + 1] = v.y, most[i + 2] = v.z, most[i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kCount; ++i)
      if (i < share && first + i < c.groups) most[i] = largest[first + i];
  }
  sample_row(block, most, first, c.group, four_at, a, row, scale, p, mass);
}

constexpr int kShort = 8192;

Chunks chunks_of(const onebit_sampling& a, void* workspace) {
  Chunks c = {};
  c.chunks = (a.vocabulary + kChunk - 1) / kChunk;
  c.group = kGroup;
  while ((a.vocabulary + c.group - 1) / c.group > kGroups) c.group *= 2;
  c.groups = (a.vocabulary + c.group - 1) / c.group;
  c.best = (mass_t*)workspace;
  c.mass = c.best + (size_t)a.rows * c.chunks;
  c.largest = (uint32_t*)(c.mass + (size_t)a.rows * c.chunks);
  return c;
}

template <int TYPE>
hipError_t launch_as(const onebit_sampling& a, void* workspace, hipStream_t stream) {
  if ((long long)a.rows * 1024 >= 1ll << 32) return hipErrorInvalidConfiguration;
  if (a.vocabulary <= kShort) {
    if (a.vocabulary <= 4096) return launch_kernel(sample_short_kernel<TYPE, 256, 4096>, dim3(a.rows), dim3(256), 0, stream, a);
    return launch_kernel(sample_short_kernel<TYPE, 512, kShort>, dim3(a.rows), dim3(512), 0, stream, a);
  }
  const Chunks c = chunks_of(a, workspace);
  // (a grid's second dimension ends at 65535: rows in parts)
  for (int first = 0; first < a.rows; first += 32768) {
    onebit_sampling part = a;
    Chunks of_part = c;
    part.rows = std::min(a.rows - first, 32768);
    const size_t size = a.logits_dtype == ONEBIT_DTYPE_F32 ? 4 : 2;
    part.logits = (const char*)a.logits + (long long)first * a.logits_stride * (long long)size;
    part.uniform += first, part.tokens += first;
    if (a.temperatures) part.temperatures += first;
    if (a.top_ps) part.top_ps += first;
    if (a.min_ps) part.min_ps += first;
    if (a.top_ks) part.top_ks += first;
    of_part.best += (size_t)first * c.chunks, of_part.mass += (size_t)first * c.chunks, of_part.largest += (size_t)first * c.groups;
    if (hipError_t status = launch_kernel(chunk_kernel<TYPE>, dim3(c.chunks, part.rows), dim3(kChunkThreads), 0, stream, part, of_part); status != hipSuccess) return status;
    if (hipError_t status = launch_kernel(sample_long_kernel<TYPE>, dim3(part.rows), dim3(kLongThreads), 0, stream, part, of_part); status != hipSuccess) return status;
  }
  return hipSuccess;
}

}  // namespace

size_t sample_workspace(const onebit_sampling& a) {
  if (a.vocabulary <= kShort) return 0;
  const Chunks c = chunks_of(a, nullptr);
  return (size_t)a.rows * (2 * sizeof(mass_t) * c.chunks + sizeof(uint32_t) * c.groups);
}

hipError_t launch_sample(const onebit_sampling& a, void* workspace, hipStream_t stream) {
  if (a.logits_dtype == ONEBIT_DTYPE_F32) return launch_as<ONEBIT_DTYPE_F32>(a, workspace, stream);
  return a.logits_dtype == ONEBIT_DTYPE_F16 ? launch_as<ONEBIT_DTYPE_F16>(a, workspace, stream) : launch_as<ONEBIT_DTYPE_BF16>(a, workspace, stream);
}

}  // namespace onebit
