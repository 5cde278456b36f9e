// Host-side argument checks shared by ops.
#pragma once

#include <ATen/core/Tensor.h>
#include <c10/util/Exception.h>

#include <initializer_list>

namespace lb {

// Every tensor lies on `like`'s device, a GPU.  Kernels take raw pointers: memory of the host or of another
// GPU would fault.  nullptr entries are skipped (arguments that were not given).
inline void check_same_device(const char* op, const at::Tensor& like,
                              std::initializer_list<const at::Tensor*> tensors) {
  TORCH_CHECK(like.is_cuda(), op, ": CUDA tensors");
  for (const at::Tensor* t : tensors)
    TORCH_CHECK(t == nullptr || t->device() == like.device(), op, ": every tensor on ",
                like.device(), ", got one on ", t->device());
}

}  // namespace lb
