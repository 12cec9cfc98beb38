// The norms around a block (onebit_decoder.h): one workgroup for each row, the row in registers from its one read to its one write.
// Bound by memory: 2048 x 8192, norm on both sides, residuals in fp32, 39.2 us for 201 MB = 5.1 TB/s, as a large copy. Small calls by the launch and one round
// of loads, so every operand of a row is requested before the first is used: 16 x 4096 3.3 us. Codes instead of y: 41.4 us for 185 MB = 4.5 TB/s, and 3.8.
// Rows that do not begin at whole vectors go by single values: 2048 x 5001 of fp16 52 us, as codes 47 (2048 x 5000: 15.7 and 19.2).
#include "onebit_codes.h"
#include "onebit_decoder_launch.h"

namespace onebit {
namespace {

constexpr int kVector = 8;

// Eight values of any type as they come from memory
struct Raw {
  u4_t low, high;
};
template <bool WHOLE>
__device__ inline Raw load_raw(const void* base, int type, long long at, int count) {
  Raw r = {};
  if (WHOLE) {
    if (type == ONEBIT_DTYPE_F32) {
      r.low = ((const u4_t*)((const float*)base + at))[0];
      r.high = ((const u4_t*)((const float*)base + at))[1];
    } else {
      r.low = *(const u4_t*)((const uint16_t*)base + at);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kVector; ++i) {
      if (i >= count) break;
      if (type == ONEBIT_DTYPE_F32) {
        const uint32_t word = ((const uint32_t*)base)[at + i];
        if (i < 4) r.low[i] = word; else r.high[i - 4] = word;
      } else {
        r.low[i / 2] |= (uint32_t)((const uint16_t*)base)[at + i] << (16 * (i % 2));
      }
    }
  }
  return r;
}
__device__ inline void widen(const Raw& raw, int type, float (&x)[kVector]) {
  if (type == ONEBIT_DTYPE_F32) {
#pragma unroll
    for (int i = 0; i < kVector; ++i) x[i] = __uint_as_float(i < 4 ? raw.low[i] : raw.high[i - 4]);
  } else if (type == ONEBIT_DTYPE_F16) {
#pragma unroll
    for (int i = 0; i < kVector; ++i) x[i] = (float)__builtin_bit_cast(h8_t, raw.low)[i];
  } else {
#pragma unroll
    for (int i = 0; i < kVector; ++i) x[i] = __uint_as_float(i % 2 ? raw.low[i / 2] & 0xffff0000u : raw.low[i / 2] << 16);
  }
}
template <bool WHOLE, bool FAR>
__device__ inline void store_row(void* base, int type, long long at, int count, const float (&x)[kVector]) {
  if (WHOLE) {
    if (type == ONEBIT_DTYPE_F32) store_values<ONEBIT_DTYPE_F32, kVector, FAR>(base, at, x);
    else if (type == ONEBIT_DTYPE_F16) store_values<ONEBIT_DTYPE_F16, kVector, FAR>(base, at, x);
    else store_values<ONEBIT_DTYPE_BF16, kVector, FAR>(base, at, x);
  } else {
#pragma unroll
    for (int i = 0; i < kVector; ++i) {
      if (i >= count) break;
      if (type == ONEBIT_DTYPE_F32) ((float*)base)[at + i] = x[i];
      else if (type == ONEBIT_DTYPE_F16) ((_Float16*)base)[at + i] = (_Float16)x[i];
      else ((__bf16*)base)[at + i] = (__bf16)x[i];
    }
  }
}

// Sum over the workgroup, the same in every thread: wavefronts in their order, so always in the same order.
__device__ inline float row_sum(float x, float* parts) {
  x = wave_sum(x);
  const int waves = blockDim.x / 64;
  if (waves == 1) return x;
  __syncthreads();  // the last sum's readers are through
  if (threadIdx.x % 64 == 0) parts[threadIdx.x / 64] = x;
  __syncthreads();
  float total = 0.f;
  for (int w = 0; w < waves; ++w) total += parts[w];
  return total;
}

// x := (x - mean) / sqrt(var + eps), or x / sqrt(mean square + eps); the variance from the differences, which one pass of sums would lose
template <int VECTORS>
__device__ inline void normalise(float (&x)[VECTORS][kVector], const onebit_norm& a, float* parts) {
  const int stride = blockDim.x * kVector;
  if (a.kind == 1) {
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < VECTORS; ++v)
#pragma unroll
      for (int i = 0; i < kVector; ++i) sum += x[v][i];  // 0 beyond the row
    const float mean = row_sum(sum, parts) / (float)a.hidden;
#pragma unroll
    for (int v = 0; v < VECTORS; ++v)
#pragma unroll
      for (int i = 0; i < kVector; ++i)
        if ((int)threadIdx.x * kVector + v * stride + i < a.hidden) x[v][i] -= mean;
  }
  float squares = 0.f;
#pragma unroll
  for (int v = 0; v < VECTORS; ++v)
#pragma unroll
    for (int i = 0; i < kVector; ++i) squares += x[v][i] * x[v][i];
  // (in 64 bits: rounded once, where fp32 would round four times what every value of the row is multiplied by)
  const float factor = (float)(1.0 / sqrt((double)row_sum(squares, parts) / a.hidden + (double)a.eps));
#pragma unroll
  for (int v = 0; v < VECTORS; ++v)
#pragma unroll
    for (int i = 0; i < kVector; ++i) x[v][i] *= factor;
}

// WHOLE: every vector is eight values at a multiple of 16 bytes. FAR: h goes past the caches. CODES: y leaves as 8-bit codes; 16 neighbouring threads, which
// are in one wavefront, hold the 128 values of a scale, and threads behind the row's end the zeros of its last group.
template <int VECTORS, bool WHOLE, bool FAR, bool CODES>
__device__ inline void norm_row(const onebit_norm& a, const onebit_codes& codes) {
  __shared__ float parts[16];
  const long long row = blockIdx.x;
  const int stride = blockDim.x * kVector;
  constexpr bool EAGER = VECTORS == 1;  // the vectors that all rows share: registers for one of each, and few rows where they are new
  Raw x[VECTORS], residual[VECTORS], weight, bias, post_weight, post_bias, gate;
  int left[VECTORS];
#pragma unroll
  for (int v = 0; v < VECTORS; ++v) {
    const int at = threadIdx.x * kVector + v * stride;
    left[v] = a.hidden - at;
    if (left[v] <= 0) continue;
    if (a.x) x[v] = load_raw<WHOLE>(a.x, a.x_dtype, row * a.x_stride + at, left[v]);
    residual[v] = load_raw<WHOLE>(a.residual, a.residual_dtype, row * a.residual_stride + at, left[v]);
  }
  auto load_gate = [&](int v) {
    return a.gate_column_stride ? load_raw<WHOLE>(a.gate, a.gate_dtype, row * a.gate_row_stride + threadIdx.x * kVector + v * stride, left[v])
                                : load_raw<false>(a.gate, a.gate_dtype, row * a.gate_row_stride, 1);
  };
  auto load_weight = [&](const void* w, int v) { return load_raw<WHOLE>(w, a.weight_dtype, threadIdx.x * kVector + v * stride, left[v]); };
  if (EAGER && left[0] > 0) {
    weight = load_weight(a.weight, 0);
    if (a.bias) bias = load_weight(a.bias, 0);
    if (a.post_weight) post_weight = load_weight(a.post_weight, 0);
    if (a.post_bias) post_bias = load_weight(a.post_bias, 0);
    if (a.gate) gate = load_gate(0);
  }
  float h[VECTORS][kVector] = {};
  if (a.x) {
#pragma unroll
    for (int v = 0; v < VECTORS; ++v)
      if (left[v] > 0) widen(x[v], a.x_dtype, h[v]);
    if (a.post_weight) {
      normalise(h, a, parts);
#pragma unroll
      for (int v = 0; v < VECTORS; ++v) {
        if (left[v] <= 0) continue;
        float w[kVector];
        widen(EAGER ? post_weight : load_weight(a.post_weight, v), a.weight_dtype, w);
#pragma unroll
        for (int i = 0; i < kVector; ++i) h[v][i] *= w[i];
        if (a.post_bias) {
          widen(EAGER ? post_bias : load_weight(a.post_bias, v), a.weight_dtype, w);
#pragma unroll
          for (int i = 0; i < kVector; ++i) h[v][i] += w[i];
        }
      }
    }
  }
#pragma unroll
  for (int v = 0; v < VECTORS; ++v) {
    if (left[v] <= 0) continue;
    float other[kVector];
    if (a.gate) {
      widen(EAGER ? gate : load_gate(v), a.gate_dtype, other);
#pragma unroll
      for (int i = 0; i < kVector; ++i) h[v][i] *= a.gate_column_stride ? other[i] : other[0];
    }
    widen(residual[v], a.residual_dtype, other);
#pragma unroll
    for (int i = 0; i < kVector; ++i) h[v][i] = (WHOLE || i < left[v]) ? a.residual_scale * other[i] + (a.x ? a.block_scale * h[v][i] : 0.f) : 0.f;
    if (a.h_out) store_row<WHOLE, FAR>(a.h_out, a.residual_dtype, row * a.h_stride + threadIdx.x * kVector + v * stride, left[v], h[v]);
  }
  normalise(h, a, parts);
#pragma unroll
  for (int v = 0; v < VECTORS; ++v) {
    if (left[v] <= 0 && !CODES) continue;
    float w[kVector];
    if (left[v] > 0) {
      widen(EAGER ? weight : load_weight(a.weight, v), a.weight_dtype, w);
#pragma unroll
      for (int i = 0; i < kVector; ++i) h[v][i] *= w[i];
      if (a.bias) {
        widen(EAGER ? bias : load_weight(a.bias, v), a.weight_dtype, w);
#pragma unroll
        for (int i = 0; i < kVector; ++i) h[v][i] += w[i];
      }
    }
    if (CODES) store_codes(codes, row, threadIdx.x * kVector + v * stride, threadIdx.x * kVector + v * stride < padded_columns(a.hidden), h[v]);
    else store_row<WHOLE, false>(a.y, a.y_dtype, row * a.y_stride + threadIdx.x * kVector + v * stride, left[v], h[v]);
  }
}
template <int VECTORS, bool WHOLE, bool FAR>
__global__ __launch_bounds__(1024) void norm_kernel(onebit_norm a) {
  norm_row<VECTORS, WHOLE, FAR, false>(a, {});
}
template <int VECTORS, bool WHOLE, bool FAR>
__global__ __launch_bounds__(1024) void norm_codes_kernel(onebit_norm a, onebit_codes codes) {
  norm_row<VECTORS, WHOLE, FAR, true>(a, codes);
}

bool whole(const void* p, long long stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % kVector == 0; }

}  // namespace

hipError_t launch_norm(const onebit_norm& a, const onebit_codes* codes, hipStream_t stream) {
  const bool vectors = a.hidden % kVector == 0 && whole(a.x, a.x ? a.x_stride : 0) && whole(a.residual, a.residual_stride) &&
                       whole(a.h_out, a.h_out ? a.h_stride : 0) && (codes || whole(a.y, a.y_stride)) && whole(a.weight, 0) && whole(a.bias, 0) &&
                       whole(a.post_weight, 0) && whole(a.post_bias, 0) && (!a.gate_column_stride || whole(a.gate, a.gate_row_stride));
  const int units = ((codes ? padded_columns(a.hidden) : a.hidden) + kVector - 1) / kVector;
  // One vector to a thread is the shortest way for few rows (16 x 4096 3.6 us, with two 4.4). Of many long rows a compute unit then holds one at a time
  // and waits for it: two vectors, half the wavefronts, and the next row under way (2048 x 8192 with a norm behind the block 51.0 us, with two 40.3).
  const int per_thread = units <= 1024 && (units < 512 || a.rows < 512) ? 1 : units <= 2048 ? 2 : 4;
  const int threads = ((units + per_thread - 1) / per_thread + 63) / 64 * 64;
  // h is read again by the next norm, with at least a projection between: of a quarter of the 256 MB of the last cache on it is written past the caches,
  // which leaves them to y (2048 x 8192, h fp32: 39.2 us for 46.3, and with the projections behind two such norms within 2 % either way;
  // 8192 x 4096 fp16 with them 319 for 324; y too past them: 40.3, and 1 to 2 % lost in what reads it; h of 16 rows: 0.6 of 14.8 us lost).
  // By itself, past the caches | through them: h of 16 MB 10.8 | 11.9 us (512 x 8192 fp32), 32 MB 19.4 | 17.6 (1024 x 8192) and 23.9 | 27.4 (4096 x 4096 fp16),
  // 48 MB 31.1 | 32.0, 64 MB 38.1 | 45.9 and 52.0 | 51.4 (8192 x 4096 fp16), 94 MB 58.2 | 60.8: below the quarter either way, and what reads h next finds it.
  const bool far = vectors && a.h_out && (long long)a.rows * a.hidden * (a.residual_dtype == ONEBIT_DTYPE_F32 ? 4 : 2) >= 64 << 20;
  auto launch = [&](auto kernel, auto codes_kernel) {
    return codes ? launch_kernel(codes_kernel, dim3(a.rows), dim3(threads), 0, stream, a, *codes) : launch_kernel(kernel, dim3(a.rows), dim3(threads), 0, stream, a);
  };
  auto launch_as = [&](auto count) {
    constexpr int kVectors = decltype(count)::value;
    return far       ? launch(norm_kernel<kVectors, true, true>, norm_codes_kernel<kVectors, true, true>)
           : vectors ? launch(norm_kernel<kVectors, true, false>, norm_codes_kernel<kVectors, true, false>)
                     : launch(norm_kernel<kVectors, false, false>, norm_codes_kernel<kVectors, false, false>);
  };
  if (per_thread == 1) return launch_as(std::integral_constant<int, 1>());
  if (per_thread == 2) return launch_as(std::integral_constant<int, 2>());
  return launch_as(std::integral_constant<int, 4>());
}

}  // namespace onebit
