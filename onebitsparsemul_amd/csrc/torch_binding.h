// What the sources of the torch binding share.
#pragma once
#include <torch/extension.h>
// PyTorch on ROCm presents its devices as type "cuda"; these are the guard and stream accessors for that.
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include "onebit_sparse_tensor.h"

using OptionalTensor = std::optional<torch::Tensor>;

inline int dtype_code(c10::ScalarType type) {
  switch (type) {
    case torch::kFloat32: return ONEBIT_DTYPE_F32;
    case torch::kFloat16: return ONEBIT_DTYPE_F16;
    case torch::kBFloat16: return ONEBIT_DTYPE_BF16;
    default: return -1;
  }
}

inline void* current_stream(const c10::Device& device) {
  return static_cast<void*>(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(device.index()).stream());
}

inline void check_status(int rc) {
  TORCH_CHECK(rc == ONEBIT_OK, "libonebitmul: ", onebit_sparse_last_error(), " (status ", rc, ")");
}

inline torch::Tensor empty_result(at::IntArrayRef sizes, c10::ScalarType type, const c10::Device& device) {
  return at::empty(sizes, at::TensorOptions().dtype(type).device(device));
}

// torch_decoder.cpp, torch_head.cpp
void bind_decoder(pybind11::module_& m);
void bind_head(pybind11::module_& m);
