// Host-side checks that several entry points share.
#pragma once

#include <torch/extension.h>

namespace ft {

// A kernel reads all its operands by address, so they have to lie on the device that it runs on.
// (A second GPU's address is valid in the first one's address space or faults there, depending on
// peer access: neither says what went wrong.)
template <class... Tensors>
inline void check_one_device(const char* op, const torch::Tensor& first, const Tensors&... rest) {
  const torch::Tensor* all[] = {&rest...};
  for (const torch::Tensor* t : all)
    TORCH_CHECK(t->device() == first.device(), op, ": all operands must be on one device, got ", first.device(), " and ",
                t->device());
}

}  // namespace ft
