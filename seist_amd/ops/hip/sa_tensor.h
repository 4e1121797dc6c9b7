// What the launchers ask of tensors.
#pragma once

#include <torch/extension.h>

namespace sa {

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
