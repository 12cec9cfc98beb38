// Host-visible launch interface of the kernels behind onebit_head.h (internal to libonebitmul). Arguments are checked.
#pragma once
#include "onebit_head.h"
#include "onebit_launch.h"

namespace onebit {

hipError_t launch_quantize_rows(const void* x, int dtype, long long x_stride, int rows, int columns, const onebit_codes& out, hipStream_t stream);

hipError_t launch_block_linear(const onebit_block_product& args, hipStream_t stream);

hipError_t launch_sample(const onebit_sampling& args, hipStream_t stream);

}  // namespace onebit
