// The instantiations of the forward row kernels for one element type (included by one file per type).
#pragma once

#include "kernels/block_norm_forward.cuh"
#include "kernels/block_norm_forward_vector.cuh"
#include "kernels/block_norm_kernels.h"

namespace afir {
namespace kernels {

template <int ELEM, int KIND, int PASS> ForwardKernel forwardKernelOf(bool vector, int nv) {
  switch (nv) {
  case 1: return vector ? blockNormForwardVectorKernel<ELEM, KIND, PASS, 1> : blockNormForwardKernel<ELEM, KIND, PASS, 1>;
  case 2: return vector ? blockNormForwardVectorKernel<ELEM, KIND, PASS, 2> : blockNormForwardKernel<ELEM, KIND, PASS, 2>;
  case 4: return vector ? blockNormForwardVectorKernel<ELEM, KIND, PASS, 4> : blockNormForwardKernel<ELEM, KIND, PASS, 4>;
  default:
    if constexpr (ELEM == kF32) return vector ? blockNormForwardVectorKernel<ELEM, KIND, PASS, 8> : blockNormForwardKernel<ELEM, KIND, PASS, 8>;
    else return nullptr;
  }
}
template <int ELEM, int KIND> ForwardKernel forwardKernelOf(int pass, bool vector, int nv) {
  if (pass == kPre) return forwardKernelOf<ELEM, KIND, kPre>(vector, nv);
  if (pass == kPost) return forwardKernelOf<ELEM, KIND, kPost>(vector, nv);
  return forwardKernelOf<ELEM, KIND, kPostPre>(vector, nv);
}
template <int ELEM> ForwardKernel forwardKernel(int kind, int pass, bool vector, int nv) {
  return kind == kLayerNorm ? forwardKernelOf<ELEM, kLayerNorm>(pass, vector, nv) : forwardKernelOf<ELEM, kRmsNorm>(pass, vector, nv);
}

} // namespace kernels
} // namespace afir
