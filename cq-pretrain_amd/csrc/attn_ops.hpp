// What the PyTorch operators of the attention layers share: checks, streams, and rows as the kernels read them.
#pragma once
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include "cqgdn.h"

namespace {

using at::Tensor;


inline hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

inline void check(int rc, const char* what) {
  if (rc == CQGDN_OK) return;
  TORCH_CHECK_VALUE(rc != CQGDN_EINVAL, what, ": ", cqgdn_last_error());
  TORCH_CHECK_NOT_IMPLEMENTED(rc != CQGDN_EUNSUPPORTED, what, ": ", cqgdn_last_error());
  TORCH_CHECK(false, what, ": ", cqgdn_last_error());
}

inline void on_one_gpu(std::initializer_list<const Tensor*> all) {
  const auto device = (*all.begin())->device();
  for (const Tensor* x : all) TORCH_CHECK_VALUE(x->device() == device, "tensors lie on different devices");
  TORCH_CHECK_VALUE(device.is_cuda(), "the hip GDN backend requires tensors on a ROCm GPU");
}

inline int dtype_code(const Tensor& x, const char* name) {
  const auto t = x.scalar_type();
  TORCH_CHECK_VALUE(t == at::kBFloat16 || t == at::kHalf, name, " must be bf16 or fp16");
  return t == at::kHalf ? CQGDN_F16 : CQGDN_BF16;
}

inline void int32_vector(const Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(x.dim() == 1 && x.scalar_type() == at::kInt, name, " must be an int32 vector");
}

// x as the kernels read rows of heads: unit stride within a head, 16-byte aligned rows
inline Tensor head_rows(const Tensor& x) {
  const bool fit = x.stride(2) == 1 && x.stride(0) % 8 == 0 && x.stride(1) % 8 == 0 &&
                   reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
  return fit ? x : x.clone(at::MemoryFormat::Contiguous);
}

}  // namespace
