// Attention over the 8-bit cache: what its kernels share (internal to libonebitmul).
//
// Mathematics: out = sum_j p_j v_j / sum_j p_j with p_j = exp2(t_j - m), t_j = log2(e) scale k_scale q . k_code_j and m the largest t so far, in
// one pass over the keys; where m grows, what is summed so far is multiplied by exp2(m_old - m). Codes are exact in fp16, and so
// is q (bf16 rows as q 2^-e; what lies below 2^-33 of a row's largest value is lost), so that the products of the matrix instructions are exact and their sums
// fp32. p_j takes its key's v_scale by its power of two beside that of the keys around it, and some powers on top, so that fp16 keeps the bits of small p_j; the
// sums follow that power exactly. What p_j v_scale comes to below 2^-32 of the largest (2^-38 where rows are few)
// counts as 0.
//
// Scores are computed as K Q^T: a lane then holds scores of one row of q (matrix column) and of the keys that the next product,
// V^T P^T, wants from it as its own operand: p goes from one matrix instruction to the next without leaving its register.
#pragma once
#include "onebit_decoder_device.h"
#include "onebit_decoder_launch.h"

namespace onebit {

constexpr float kLog2E = 1.44269504088896340736f;

// Four codes of a word as fp16, exact. e4m3 by the conversion instruction; int8: the byte plus 128 as the low byte of 1024 + n, minus 1152.
template <int CODE>
__device__ inline void codes_to_f16(uint32_t word, h2_t& low, h2_t& high) {
  if constexpr (CODE == ONEBIT_CODE_E4M3) {
    low = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.f, false));
    high = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.f, true));
  } else {
    const uint32_t shifted = word ^ 0x80808080u;
    const h2_t offset = {(_Float16)1152.f, (_Float16)1152.f};
    low = __builtin_bit_cast(h2_t, __builtin_amdgcn_perm(0x64646464u, shifted, 0x04010400u)) - offset;
    high = __builtin_bit_cast(h2_t, __builtin_amdgcn_perm(0x64646464u, shifted, 0x04030402u)) - offset;
  }
}
template <int CODE>
__device__ inline h8_t codes_to_f16(uint32_t first, uint32_t second) {
  h2_t a, b, c, d;
  codes_to_f16<CODE>(first, a, b);
  codes_to_f16<CODE>(second, c, d);
  return h8_t{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// Words of four tokens' codes at four dims -> words of four dims' codes of the four tokens
__device__ inline void transpose_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t (&out)[4]) {
  const uint32_t ab_low = __builtin_amdgcn_perm(b, a, 0x05010400u), ab_high = __builtin_amdgcn_perm(b, a, 0x07030602u);
  const uint32_t cd_low = __builtin_amdgcn_perm(d, c, 0x05010400u), cd_high = __builtin_amdgcn_perm(d, c, 0x07030602u);
  out[0] = __builtin_amdgcn_perm(cd_low, ab_low, 0x05040100u);
  out[1] = __builtin_amdgcn_perm(cd_low, ab_low, 0x07060302u);
  out[2] = __builtin_amdgcn_perm(cd_high, ab_high, 0x05040100u);
  out[3] = __builtin_amdgcn_perm(cd_high, ab_high, 0x07060302u);
}

// The larger of each lane's value and those of the lanes 16, 32 and 48 further on
__device__ inline float max_over_16(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float sum_over_16(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ inline float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // -126 <= e <= 127
__device__ inline float power_or_zero(int e) { return e < -126 ? 0.f : power_of_two(e); }
// Exponent of a normal magnitude (a NaN and infinities: 128)
__device__ inline int exponent_of(uint32_t magnitude_bits) { return (int)(magnitude_bits >> 23) - 127; }

// What takes a v_scale's part in exponents: one below 2^-100 is as good as 0, one that is not finite is dealt with apart. The largest finite value makes
// scales below 2^122 (over 127); an exponent of theirs has room for its neighbours here, and for its negative.
__device__ inline float usable_scale(float scale) {
  return magnitude(scale) >= 0x7f800000u ? 0x1p-100f : fminf(fmaxf(scale, 0x1p-100f), 0x1.fffffep121f);
}
// The exponent that the sums stand in: that of the keys' v_scale at hand, followed where it grows or falls by more than a few, for fp16 to keep the
// bits of small p beside it. Never further below the largest so far than fp32 has room for. It is one for all rows, also for those that do not see the
// largest: their sums stand as far below it as fp32 reaches.
struct Exponent {
  int now = -100, largest = -100;  // -100: nothing yet but what is as good as 0
  // The power of two that the sums take on.
  __device__ float follow(int power) {
    if (power <= now && power >= now - 6) return 1.f;
    largest = max(largest, power);
    const int next = max(power, max(largest - 60, -99));
    const float factor = now == -100 ? 0.f : power_or_zero(now - next);
    now = next;
    return factor;
  }
};

__device__ inline float lane_value(float x, int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), lane)); }

// Eight values of a row of q: the largest magnitude, and as fp16 times `factor` (a power of two; not used on fp16)
__device__ inline uint32_t magnitude_bf16(u4_t q) {
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) most = max(most, max((q[i] << 16) & 0x7fff0000u, q[i] & 0x7fff0000u));
  return most;
}
__device__ inline h8_t q_to_f16(u4_t raw, int dtype, float factor) {
  if (dtype == ONEBIT_DTYPE_F16) return __builtin_bit_cast(h8_t, raw);
  h8_t r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[2 * i] = (_Float16)(__uint_as_float(raw[i] << 16) * factor);
    r[2 * i + 1] = (_Float16)(__uint_as_float(raw[i] & 0xffff0000u) * factor);
  }
  return r;
}

// The pages of a sequence from entry `first` of its table on, one to a lane
struct Window {
  int first;
  int page;  // -1: none
  float k_scale, v_scale;
};
__device__ inline Window load_pages(int entry, int width, const int* table, const onebit_cache& cache) {
  const int own = entry + (int)(threadIdx.x % 64);
  Window window = {entry, own < width ? table[own] : -1, 0.f, 0.f};
  if (window.page >= cache.pages) window.page = -1;
  return window;
}
// Drops the window's pages behind entry `last`.
__device__ inline void drop_pages(Window& window, int last) {
  if (window.first + (int)(threadIdx.x % 64) > last) window.page = -1;
}
__device__ inline void load_scales(Window& window, const onebit_cache& cache, int head) {
  window.k_scale = window.v_scale = 0.f;
  if (window.page >= 0) {
    const long long at = (long long)window.page * cache.kv_heads + head;
    window.k_scale = cache.k_scale[at];
    window.v_scale = cache.v_scale[at];
  }
}
// token and head of the key/value head of a row of q, `step` rows behind the first of a tile
struct Rows {
  int token, head;  // of the tile's first row
};
__device__ inline Rows first_row(int row, int group) { return row == 0 ? Rows{0, 0} : Rows{row / group, row % group}; }
__device__ inline Rows behind(Rows first, int step, const AttentionArgs& args) {
  // exact: numbers below group + 256, whose product with group (at most 32768) is below 2^32
  const uint32_t n = first.head + step, tokens = args.group == 1 ? n : __umulhi(n, args.group_inverse);
  return {first.token + (int)tokens, (int)(n - tokens * args.group)};
}

}  // namespace onebit
