// What the torch binding files share: argument helpers, the device error word, the current stream.
#pragma once
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <cstdlib>
#include <cstring>
#include <limits>
#include <string>
#include <vector>

#include "kernels.h"

#define DFL_CHECK_RC(rc, what) TORCH_CHECK((rc) == 0, what, " launch failed with status ", (rc))

inline void check_bf16_cuda(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.scalar_type() == at::kBFloat16, name, " must be bfloat16");
}

inline void check_rowmajor(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.dim() == 2, name, " must be 2-D");
  TORCH_CHECK(t.stride(1) == 1, name, " must have a unit inner stride");
}

// Per-device 4-int error word (see common.cuh).
inline at::Tensor& error_buffer(int device) {
  static at::Tensor bufs[16];
  TORCH_CHECK(device >= 0 && device < 16, "device index out of range");
  if (!bufs[device].defined()) {
    bufs[device] = at::zeros({4}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, device));
  }
  return bufs[device];
}

inline int* err_ptr() {
  int dev = c10::cuda::current_device();
  return error_buffer(dev).data_ptr<int>();
}

inline cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

inline const void* opt_ptr(const c10::optional<at::Tensor>& t) {
  return (t.has_value() && t->defined()) ? t->data_ptr() : nullptr;
}

// at::empty on t's device without the dispatcher (a microsecond of a small call).
inline at::Tensor new_like(const at::Tensor& t, at::IntArrayRef sizes, at::ScalarType dtype) {
  return at::detail::empty_cuda(sizes, dtype, t.device(), c10::nullopt);
}

inline int dtype_code(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return kDtypeF32;
    case at::kBFloat16: return kDtypeBf16;
    case at::kHalf: return kDtypeF16;
    default: TORCH_CHECK_VALUE(false, name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
  }
}

inline const at::Tensor* given(const c10::optional<at::Tensor>& t) { return t.has_value() && t->defined() ? &*t : nullptr; }

// No wrapper among these (function transforms such as vmap, fake tensors) and no forward-mode tangent.
inline bool plain_tensors(std::initializer_list<const at::Tensor*> tensors) {
  constexpr c10::DispatchKeySet wrappers({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched,
                                          c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize});
  for (const at::Tensor* t : tensors)
    if (t && (t->key_set().has_any(wrappers) || t->_fw_grad(0).defined())) return false;
  return true;
}

// Tensors that a kernel can be given in place of a differentiable torch operation: none asks for gradients or carries a
// forward-mode tangent, and none is a wrapper (function transforms such as vmap, fake tensors).
inline bool kernel_tensors(std::initializer_list<const at::Tensor*> tensors) {
  if (at::GradMode::is_enabled())
    for (const at::Tensor* t : tensors)
      if (t && t->requires_grad()) return false;
  return plain_tensors(tensors);
}
