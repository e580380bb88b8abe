// What the operator registrations share: tensor descriptors, stream and error handling.
#pragma once

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <initializer_list>

#include "relation_lm_hip.h"

namespace {

int32_t dtype_code(at::ScalarType s) {
  switch (s) {
    case at::kFloat: return RLM_F32;
    case at::kBFloat16: return RLM_BF16;
    case at::kHalf: return RLM_F16;
    case at::kInt: return RLM_I32;
    case at::kLong: return RLM_I64;
    default: return -1;
  }
}

rlm_tensor desc(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.defined(), name, ": tensor is undefined");
  TORCH_CHECK(t.dim() <= RLM_MAX_DIMS, name, ": at most ", RLM_MAX_DIMS, " dims supported");
  const int32_t code = dtype_code(t.scalar_type());
  TORCH_CHECK(code >= 0, name, ": unsupported dtype ", t.scalar_type());
  rlm_tensor d{};
  d.data = t.data_ptr();
  d.dtype = code;
  d.ndim = static_cast<int32_t>(t.dim());
  for (int64_t i = 0; i < t.dim(); ++i) {
    d.shape[i] = t.size(i);
    d.stride[i] = t.stride(i);
  }
  return d;
}

// All tensors must live on one ROCm device; returns its current stream.
hipStream_t device_stream(const char* op, std::initializer_list<const at::Tensor*> tensors) {
  const at::Tensor* first = *tensors.begin();
  TORCH_CHECK(first->is_cuda(), op, ": relation_lm HIP ops need tensors on a ROCm device, got ",
              first->device());
  for (const at::Tensor* t : tensors) {
    if (!t->defined()) continue;
    TORCH_CHECK(t->is_cuda() && t->device() == first->device(), op,
                ": all tensors must be on ", first->device(), ", found one on ", t->device());
  }
  return c10::hip::getCurrentHIPStream(first->device().index()).stream();
}

void check(hipError_t err, const char* op) {
  TORCH_CHECK(err == hipSuccess, op, " failed (hipError ", static_cast<int>(err), "): ",
              rlm_last_error());
}

at::TensorOptions f32(const at::Tensor& like) { return like.options().dtype(at::kFloat); }
at::TensorOptions i32(const at::Tensor& like) { return like.options().dtype(at::kInt); }

}  // namespace
