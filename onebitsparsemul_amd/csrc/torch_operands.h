// Operands of the decoder's operators as torch tensors: checks, whether two of them meet in memory, rows.
#pragma once
#include "torch_binding.h"

#include "onebit_head.h"

#include <algorithm>
#include <vector>

inline void check_gpu(const torch::Tensor& t, const char* name, const c10::Device& device) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.device() == device, name, " must live on ", device, ", got ", t.device());
}

// A contiguous vector or matrix of the call's plan, as it is
inline void check_table(const torch::Tensor& t, const char* name, c10::ScalarType type, int64_t dims, const c10::Device& device) {
  check_gpu(t, name, device);
  TORCH_CHECK_TYPE(t.scalar_type() == type, name, " must be ", type, ", got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() == dims && t.is_contiguous() && !t.is_neg(), name, " must be contiguous with ", dims, " dimensions, got shape ", t.sizes());
}

// The bytes from a tensor's first element to its last
inline std::pair<const char*, const char*> extent(const torch::Tensor& t) {
  int64_t last = 0;
  for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
  const char* const first = (const char*)t.data_ptr();
  return {first, first + (last + 1) * t.element_size()};
}
// Whether sum of x_i step_i = distance for some x_i from -below_i to above_i; true also where there are many to try. Steps from the largest on.
struct Step {
  int64_t step, below, above;
};
inline bool reaches(const std::vector<Step>& steps, size_t from, int64_t distance) {
  if (from == steps.size()) return distance == 0;
  int64_t low = 0, high = 0;  // of the others
  for (size_t i = from + 1; i < steps.size(); ++i) low -= steps[i].step * steps[i].below, high += steps[i].step * steps[i].above;
  const Step s = steps[from];
  int tries = 0;
  for (int64_t x = std::max(-s.below, (distance - high) / s.step - 1); x <= std::min(s.above, (distance - low) / s.step + 1); ++x)
    if (++tries > 8 || reaches(steps, from + 1, distance - x * s.step)) return true;
  return false;
}
// Whether two tensors may have memory in common: exactly for views that go through it in the same steps, else by their extents.
inline bool may_meet(const torch::Tensor& a, const torch::Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  const auto one = extent(a), other = extent(b);
  if (one.second <= other.first || other.second <= one.first) return false;
  const int64_t distance = other.first - one.first, size = a.element_size();
  if (a.dim() != b.dim() || b.element_size() != size || distance % size) return true;
  std::vector<Step> steps;
  for (int64_t i = 0; i < a.dim(); ++i) {
    if (a.size(i) > 1 && b.size(i) > 1 && a.stride(i) != b.stride(i)) return true;
    const int64_t step = a.size(i) > 1 ? a.stride(i) : b.stride(i);
    if (step != 0 && (a.size(i) > 1 || b.size(i) > 1)) steps.push_back({step, b.size(i) - 1, a.size(i) - 1});
  }
  std::sort(steps.begin(), steps.end(), [](const Step& x, const Step& y) { return x.step > y.step; });
  return reaches(steps, 0, distance / size);
}
// (rows, hidden) from (..., hidden), a view or a copy
inline torch::Tensor rows_of(const torch::Tensor& t, int64_t hidden) {
  torch::Tensor r = t.dim() == 2 ? t : t.reshape({-1, hidden});
  return (r.stride(1) == 1 || hidden == 1) && !r.is_neg() ? r : r.resolve_neg().clone(at::MemoryFormat::Contiguous);
}

// Codes and scales of rows of `sizes` values (onebit_head.h), the rows one behind the other
inline std::tuple<torch::Tensor, torch::Tensor> empty_codes(at::IntArrayRef sizes, const c10::Device& device) {
  std::vector<int64_t> shape = sizes.vec();
  const int64_t groups = (shape.back() + ONEBIT_CODE_GROUP - 1) / ONEBIT_CODE_GROUP;
  shape.back() = groups * ONEBIT_CODE_GROUP;
  torch::Tensor codes = empty_result(shape, torch::kFloat8_e4m3fn, device);
  shape.back() = groups;
  return {codes, empty_result(shape, torch::kFloat32, device)};
}
inline onebit_codes codes_of(const torch::Tensor& codes, const torch::Tensor& scales) {
  const bool rows = codes.dim() == 2;  // else consecutive
  return {codes.data_ptr(), (float*)scales.data_ptr(), rows ? codes.size(0) > 1 ? codes.stride(0) : 0 : codes.size(-1),
          rows ? scales.size(0) > 1 ? scales.stride(0) : 0 : scales.size(-1)};
}
