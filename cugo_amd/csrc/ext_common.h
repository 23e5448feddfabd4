// What the binding's source files (torch_ext.cpp, learner_ext.cpp, paged_ext.cpp) share: checks of tensors with
// the reference's messages (torch50_ext.cu:26-51), the current stream, outputs.
#ifndef CUGO_EXT_COMMON_H_
#define CUGO_EXT_COMMON_H_

#include <torch/extension.h>

// PyTorch-ROCm keeps torch's device type "cuda" for HIP devices; these are its native
// HIP guard and stream accessors for that device type.
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <cstdint>
#include <vector>

#include "../../include/cugo_hip.h"

namespace cugo_ext {

inline void check_1d(const torch::Tensor& t, at::ScalarType dtype, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  TORCH_CHECK(t.dim() == 1, name, " must be one-dimensional");
  TORCH_CHECK(t.scalar_type() == dtype, name, " has the wrong dtype");
}

inline void check_same_device(const torch::Tensor& a, const torch::Tensor& b, const char* an,
                       const char* bn) {
  TORCH_CHECK(a.device() == b.device(), an, " and ", bn, " must be on the same CUDA device");
}

inline void check_call(int rc, const char* op) {
  TORCH_CHECK(rc == 0, "cugo_hip ", op, " failed with code ", rc);
}

inline hipStream_t stream() { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }

using DeviceGuard = c10::hip::HIPGuardMasqueradingAsCUDA;

inline torch::TensorOptions on(const torch::Tensor& t, at::ScalarType dtype) {
  return torch::TensorOptions().device(t.device()).dtype(dtype);
}

// `out` if given (a contiguous tensor of `dtype` and `shape` on like's device: a caller's
// buffer the kernel writes into), else a new tensor.
inline torch::Tensor out_or_new(const c10::optional<torch::Tensor>& out, std::vector<int64_t> shape,
                         at::ScalarType dtype, const torch::Tensor& like, const char* name) {
  if (!out.has_value()) return torch::empty(shape, on(like, dtype));
  TORCH_CHECK(out->is_contiguous() && out->scalar_type() == dtype &&
                  out->sizes() == at::IntArrayRef(shape),
              name, " must be a contiguous ", c10::toString(dtype), " tensor of shape ", shape);
  check_same_device(like, *out, "input", name);
  return *out;
}

inline uint8_t* u8p(const torch::Tensor& t) { return reinterpret_cast<uint8_t*>(t.data_ptr()); }

// learner_ext.cpp: the learner's operations, added to the module.
void bind_learner(pybind11::module_& m);

// paged_ext.cpp: the paged cache's operations, added to the module.
void bind_paged(pybind11::module_& m);

}  // namespace cugo_ext

#endif  // CUGO_EXT_COMMON_H_
