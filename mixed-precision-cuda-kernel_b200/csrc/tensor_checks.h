// Checks of tensors and outputs from torch's allocator, shared by the sources of the `quant_cuda` module.
#pragma once

#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include "cherryq.h"

namespace checks {

using OptTensor = c10::optional<torch::Tensor>;

inline void check_status(int rc, const char* what) {
  if (rc == CQ_OK) return;
  TORCH_CHECK(rc != CQ_ERR_CUDA, what, ": CUDA error ", cq_last_cuda_error());
  TORCH_CHECK(false, what, ": ", cq_strerror(rc));
}

inline void check_tensor(const torch::Tensor& t, const char* name, c10::ScalarType dtype, const c10::Device& device) {
  TORCH_CHECK(t.defined() && t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.scalar_type() == dtype, name, " must have dtype ", c10::toString(dtype), ", got ", c10::toString(t.scalar_type()));
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  TORCH_CHECK(t.device() == device, name, " is on ", t.device(), ", not on ", device);
}

inline bool aligned16(const torch::Tensor& t) { return ((uintptr_t)t.const_data_ptr() & 15) == 0; }

inline void check_mask(int64_t window, int64_t sinks) {
  TORCH_CHECK(window >= 0 && window <= INT32_MAX && sinks >= 0 && sinks <= INT32_MAX, "window and sinks must not be negative");
}

inline const long long* whole_numbers(const torch::Tensor& t, const char* name, int64_t n, const c10::Device& device) {
  check_tensor(t, name, torch::kInt64, device);
  TORCH_CHECK(t.numel() == n, name, " must have ", n, " entries");
  return (const long long*)t.const_data_ptr();
}

// An output or workspace, straight from the allocator: short calls are bound by the host, and a trip through the dispatcher for
// each of them costs more than the rest of a call.  (Not where a dispatch mode watches.)
inline torch::Tensor fresh_on(const c10::Device& device, c10::IntArrayRef shape, c10::ScalarType type) {
  if (c10::impl::TorchDispatchModeTLS::any_modes_set()) return torch::empty(shape, torch::TensorOptions().device(device).dtype(type));
  return at::detail::empty_cuda(shape, type, device, c10::nullopt);
}

}  // namespace checks
