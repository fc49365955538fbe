// The instantiations of the gradient row kernels for one element type (included by one file per type).
#pragma once

#include "kernels/block_norm_grad.cuh"
#include "kernels/block_norm_kernels.h"

namespace afir {
namespace kernels {

template <int ELEM, int KIND, int PASS> GradKernel gradKernelOf(int nv) {
  switch (nv) {
  case 1: return blockNormGradKernel<ELEM, KIND, PASS, 1>;
  case 2: return blockNormGradKernel<ELEM, KIND, PASS, 2>;
  case 4: return blockNormGradKernel<ELEM, KIND, PASS, 4>;
  default:
    if constexpr (ELEM == kF32) return blockNormGradKernel<ELEM, KIND, PASS, 8>;
    else return nullptr;
  }
}
template <int ELEM> GradKernel gradKernel(int kind, int pass, int nv) {
  if (kind == kLayerNorm)
    return pass == kPre ? gradKernelOf<ELEM, kLayerNorm, kPre>(nv) : pass == kPost ? gradKernelOf<ELEM, kLayerNorm, kPost>(nv) : gradKernelOf<ELEM, kLayerNorm, kPostPre>(nv);
  return pass == kPre ? gradKernelOf<ELEM, kRmsNorm, kPre>(nv) : pass == kPost ? gradKernelOf<ELEM, kRmsNorm, kPost>(nv) : gradKernelOf<ELEM, kRmsNorm, kPostPre>(nv);
}
} // namespace kernels
} // namespace afir
