// The matrix product of 8-bit codes with a scale for each 128 (onebit_head.h).
//
// Codes go into the matrix instructions as fp16, exactly, whose products are exact and whose sums are fp32 (v_mfma_f32_16x16x32_f16: 9e-9 off over a group of 128
// normal values; those of the 8-bit instructions drop what lies 2^-14 below the largest product of a few neighbours, 1.5e-5). The sum of a group, from 0 on, times the
// product of the two scales is added to the sums in fp32. The weight is the matrix operand A, the tokens are B's columns: a lane then holds four neighbouring rows of y of
// one token, so that its scale is one register, the weight's is the same for all lanes, and y is written in vectors.
#include "onebit_codes.h"
#include "onebit_head_launch.h"

namespace onebit {
namespace {

// A lane's 32 codes of a group as fp16
struct Values {
  h8_t v[4];
};
__device__ inline Values load32(const uint8_t* p) {
  const u4_t low = ((const u4_t*)p)[0], high = ((const u4_t*)p)[1];
  return {codes_to_f16<ONEBIT_CODE_E4M3>(low.x, low.y), codes_to_f16<ONEBIT_CODE_E4M3>(low.z, low.w), codes_to_f16<ONEBIT_CODE_E4M3>(high.x, high.y),
          codes_to_f16<ONEBIT_CODE_E4M3>(high.z, high.w)};
}

__device__ inline f4_t multiply(const Values& a, const Values& b) {
  f4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i) sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v[i], b.v[i], sum, 0, 0, 0);
  return sum;
}

__device__ inline float value_at(const void* base, int type, long long at) {
  if (type == ONEBIT_DTYPE_F32) return ((const float*)base)[at];
  return type == ONEBIT_DTYPE_F16 ? (float)((const _Float16*)base)[at] : (float)((const __bf16*)base)[at];
}

// A wavefront: 16 rows of the weight, 16 tokens, operands straight from memory.
template <int TYPE>
__global__ __launch_bounds__(256) void product_kernel(onebit_block_product p) {
  const int lane = threadIdx.x % 64, n = lane % 16, quarter = lane / 16;
  const int first_row = (blockIdx.x * 4 + threadIdx.x / 64) * 16, first_token = blockIdx.y * 16;
  if (first_row >= p.rows) return;
  const int token = min(first_token + n, p.tokens - 1), row = min(first_row + n, p.rows - 1), groups = p.columns / ONEBIT_CODE_GROUP;
  const uint8_t* w = (const uint8_t*)p.weight.codes + row * p.weight.row_stride + quarter * 32;
  const uint8_t* x = (const uint8_t*)p.x.codes + token * p.x.row_stride + quarter * 32;
  const float* w_scale = p.weight.scales + first_row / ONEBIT_CODE_GROUP * p.weight.scale_stride;
  const float* x_scale = p.x.scales + token * p.x.scale_stride;
  f4_t sum = {0.f, 0.f, 0.f, 0.f};
  for (int g = 0; g < groups; ++g) {
    const f4_t part = multiply(load32(w + g * ONEBIT_CODE_GROUP), load32(x + g * ONEBIT_CODE_GROUP));
    const float scale = w_scale[g] * x_scale[g];
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] += scale * part[i];
  }
  if (first_token + n >= p.tokens) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = first_row + quarter * 4 + i;
    if (at >= p.rows) return;
    const float y[1] = {p.bias ? sum[i] + value_at(p.bias, p.bias_dtype, at) : sum[i]};
    store_values<TYPE, 1>(p.y, token * p.y_stride + at, y);
  }
}

template <int TYPE>
hipError_t launch_as(const onebit_block_product& p, hipStream_t stream) {
  return launch_kernel(product_kernel<TYPE>, dim3((p.rows + 63) / 64, (p.tokens + 15) / 16), dim3(256), 0, stream, p);
}

}  // namespace

hipError_t launch_block_linear(const onebit_block_product& p, hipStream_t stream) {
  if (p.y_dtype == ONEBIT_DTYPE_F32) return launch_as<ONEBIT_DTYPE_F32>(p, stream);
  return p.y_dtype == ONEBIT_DTYPE_F16 ? launch_as<ONEBIT_DTYPE_F16>(p, stream) : launch_as<ONEBIT_DTYPE_BF16>(p, stream);
}

}  // namespace onebit
