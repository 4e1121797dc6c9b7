// What the launchers ask of tensors.
#pragma once

#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

namespace sa {

// Whether a call is recorded, or its results are put in place by a mode: a
// tracer sees what is allocated here and not what is launched, and under such
// a mode that has no memory.
inline bool recorded() {
  using Modes = c10::impl::TorchDispatchModeTLS;
  using Key = c10::impl::TorchDispatchModeKey;
  return torch::jit::tracer::isTracing() ||
         (Modes::any_modes_set() && (Modes::get_mode(Key::FAKE) ||
                                     Modes::get_mode(Key::PROXY) ||
                                     Modes::get_mode(Key::FUNCTIONAL)));
}

// whether t's type computes in Python, as that of fake tensors, outside of
// their mode too
inline bool stands_in(const at::Tensor& t) {
  return t.key_set().has(c10::DispatchKey::Python);
}
inline bool stands_in(const c10::optional<at::Tensor>& t) {
  return t.has_value() && stands_in(*t);
}

// Where a tensor's values are. Tensors that only stand for others (fake and
// functional ones, and what is allocated while a mode puts those in place)
// have a null pointer, which a kernel would read or write all the same.
template <typename T = void>
T* memory_of(const at::Tensor& t) {
  void* p = t.data_ptr();
  TORCH_CHECK(p != nullptr || t.numel() == 0,
              "a tensor of ", t.sizes(), " has no memory to compute with");
  return (T*)p;
}

// whether forward mode carries a derivative along with t: the kernels would
// drop it
inline bool has_tangent(const at::Tensor& t) {
  return t.defined() && t._fw_grad(/*level=*/0).defined();
}

}  // namespace sa
