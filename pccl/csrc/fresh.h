// New tensors for results and workspaces of small calls.
#pragma once
#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>

namespace pccl {

// at::empty on a device without the dispatcher's way there, which small calls feel: on the host a backward call of attention takes 11.8
// us (with at::empty 12.9), one of the query/key norms 9.9 (11.4).  All of the memory is written by the call.
inline at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}

}  // namespace pccl
