// What the native call paths of the paged cache and of the operators around attention share (torch_cache.cpp, torch_decode.cpp): outputs from
// torch's allocator, checks of tensors, streams.
#pragma once
#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAStream.h>

#include <initializer_list>
#include <optional>

#include "chill_b200.h"

namespace chill_torch {
using at::Tensor;

// Without the dispatcher: 0.7 us instead of 1.1, and a call makes up to three.
inline Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) { return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt); }

// A tensor that something looks in on (a subclass with its own dispatch, a transform), or of which the memory is not the numbers: a sign still to be applied (z.conj().imag),
// zeros that were never written.  The dispatcher ops serve it.
inline bool watched(std::initializer_list<const Tensor*> tensors, const std::optional<Tensor>& one_more = std::nullopt, const std::optional<Tensor>& another = std::nullopt) {
  constexpr c10::DispatchKeySet kOthers = c10::python_ks | c10::functorch_transforms_ks | c10::DispatchKeySet({c10::DispatchKey::Negative, c10::DispatchKey::ZeroTensor});
  auto looked_at = [](const Tensor& t) { return t.unsafeGetTensorImpl()->key_set().has_any(kOthers); };
  for (const Tensor* t : tensors)
    if (looked_at(*t)) return true;
  return (one_more.has_value() && looked_at(*one_more)) || (another.has_value() && looked_at(*another));
}

inline void* current_stream(const Tensor& t) { return (void*)c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

inline void set_strides(int64_t* dst, const Tensor& t) {
  for (int64_t d = 0; d < t.dim(); ++d) dst[d] = t.stride(d);
}

inline int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return CHILL_F32;
    case at::kHalf: return CHILL_F16;
    case at::kBFloat16: return CHILL_BF16;
    default: return -1;
  }
}

// An int32 tensor of these sizes on the device of `like`, contiguous.
inline bool ints(const Tensor& t, std::initializer_list<int64_t> sizes, const Tensor& like) {
  return t.scalar_type() == at::kInt && t.sizes() == at::IntArrayRef(sizes) && t.is_contiguous() && t.device() == like.device();
}

// The C ABI takes 32-bit sizes.
inline bool fit(const Tensor& t) {
  for (const int64_t n : t.sizes())
    if (n > INT32_MAX) return false;
  return true;
}

inline bool table_ok(const Tensor& table) {
  return fit(table) && table.scalar_type() == at::kInt && table.dim() == 2 && table.size(0) > 0 && table.size(1) > 0 && table.is_cuda() && table.stride(1) == 1 &&
         (table.size(0) == 1 || table.stride(0) >= table.size(1));
}

// Gradients asked for, or a tangent carried along (forward mode, which no_grad leaves on).
inline bool wants_grad(std::initializer_list<const Tensor*> tensors) {
  const bool backward = at::GradMode::is_enabled(), forward = c10::AutogradState::get_tls_state().get_fw_grad_mode();
  for (const Tensor* t : tensors)
    if ((backward && t->requires_grad()) || (forward && t->_fw_grad(/*level=*/0).defined())) return true;
  return false;
}

// Changed in place: autograd looks at a tensor's version where it saved one.  (Inference tensors have none.)
inline void changed(std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

inline const int32_t* optional_ints(const std::optional<Tensor>& t) { return t.has_value() ? t->const_data_ptr<int32_t>() : nullptr; }

template <class F>
F pointer(uint64_t address) {
  return reinterpret_cast<F>(static_cast<uintptr_t>(address));
}

}  // namespace chill_torch
