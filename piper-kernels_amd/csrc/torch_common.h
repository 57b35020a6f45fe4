// What the torch kernels of libpiper_torch.so share.
#pragma once

#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/library.h>

#include "piper_mi355x.h"

namespace piper_torch {

inline void check(int status, const char* what) {
  TORCH_CHECK(status == PIPER_OK, what, " failed (status ", status, "): ", piper_last_error());
}

inline int32_t dtype_code(at::ScalarType type) {
  TORCH_CHECK(type == at::kHalf || type == at::kBFloat16, "piper_kernels: tensors must use float16 or bfloat16, got ", type);
  return type == at::kBFloat16 ? PIPER_BFLOAT16 : PIPER_FLOAT16;
}

inline int32_t dtype_code(const at::Tensor& t) { return dtype_code(t.scalar_type()); }

// Any [B, H, S, D] view whose rows are 16-byte aligned is read in place (the strides of axes of size 1 do
// not count); anything else is copied.  A copy, not contiguous(): that keeps a contiguous view as it is, also
// one that starts between two 16-byte boundaries.
inline at::Tensor native_input(const at::Tensor& t) {
  bool in_place = (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15u) == 0 && t.stride(3) == 1;
  for (int64_t axis = 0; axis < 3; ++axis) in_place = in_place && (t.size(axis) == 1 || t.stride(axis) % 8 == 0);
  return in_place ? t : t.clone(at::MemoryFormat::Contiguous);
}

inline piper_tensor tensor_arg(const at::Tensor& t) {
  const auto stride = [&](int64_t axis) { return t.size(axis) == 1 ? 0 : t.stride(axis); };
  return piper_tensor{t.const_data_ptr(), stride(0), stride(1), stride(2)};
}

// Registers the cache operators' kernels (csrc/torch_cache.cpp).
void register_cache_kernels(torch::Library& library);

}  // namespace piper_torch
