// The instantiations of the grad row kernel for one element type (included by one file per type).
#pragma once

#include "kernels/block_norm_grad.cuh"
#include "kernels/block_norm_kernels.h"

namespace afir {
namespace kernels {

template <int ELEM, int KIND, int PASS> GradKernel gradKernelOf(bool vector, int nv) {
  constexpr int V = ElemOf<ELEM>::kVec;
  if (!vector) return nv <= kScalarSmall ? blockNormGradKernel<ELEM, KIND, PASS, 1, kScalarSmall> : blockNormGradKernel<ELEM, KIND, PASS, 1, kScalarLarge>;
  switch (nv) {
  case 1: return blockNormGradKernel<ELEM, KIND, PASS, V, 1>;
  case 2: return blockNormGradKernel<ELEM, KIND, PASS, V, 2>;
  case 4: return blockNormGradKernel<ELEM, KIND, PASS, V, 4>;
  default:
    if constexpr (ELEM == kF32) return blockNormGradKernel<ELEM, KIND, PASS, V, 8>;
    else return nullptr;
  }
}
template <int ELEM, int KIND> GradKernel gradKernelOf(int pass, bool vector, int nv) {
  if (pass == kPre) return gradKernelOf<ELEM, KIND, kPre>(vector, nv);
  if (pass == kPost) return gradKernelOf<ELEM, KIND, kPost>(vector, nv);
  return gradKernelOf<ELEM, KIND, kPostPre>(vector, nv);
}
template <int ELEM> GradKernel gradKernel(int kind, int pass, bool vector, int nv) {
  return kind == kLayerNorm ? gradKernelOf<ELEM, kLayerNorm>(pass, vector, nv) : gradKernelOf<ELEM, kRmsNorm>(pass, vector, nv);
}

} // namespace kernels
} // namespace afir
