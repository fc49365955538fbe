// The instantiations of the gradient row kernels for one element type (included by one file per type).
#pragma once

#include "kernels/block_norm_grad.cuh"
#include "kernels/block_norm_grad_vector.cuh"
#include "kernels/block_norm_kernels.h"

namespace afir {
namespace kernels {

// Vectors without rows fetched ahead: rows too wide for two of them in shared memory.
template <int ELEM, int KIND, int PASS> GradKernel gradKernelOf(bool vector, int nv) {
  constexpr int V = ElemOf<ELEM>::kVec;
  if (!vector) return nv <= kScalarSmall ? blockNormGradKernel<ELEM, KIND, PASS, 1, kScalarSmall> : blockNormGradKernel<ELEM, KIND, PASS, 1, kScalarLarge>;
  if (nv <= 4) return blockNormGradKernel<ELEM, KIND, PASS, V, 4>;
  if constexpr (ELEM == kF32) return blockNormGradKernel<ELEM, KIND, PASS, V, 8>;
  else return nullptr;
}
template <int ELEM, int KIND, int PASS> GradAheadKernel gradAheadKernelOf(int nv) {
  switch (nv) {
  case 1: return blockNormGradVectorKernel<ELEM, KIND, PASS, 1>;
  case 2: return blockNormGradVectorKernel<ELEM, KIND, PASS, 2>;
  case 4:
    if constexpr (ELEM == kF32) return blockNormGradVectorKernel<ELEM, KIND, PASS, 4>;
    else return nullptr;
  default: return nullptr;
  }
}
template <int ELEM> GradKernel gradKernel(int kind, int pass, bool vector, int nv) {
  if (kind == kLayerNorm)
    return pass == kPre ? gradKernelOf<ELEM, kLayerNorm, kPre>(vector, nv) : pass == kPost ? gradKernelOf<ELEM, kLayerNorm, kPost>(vector, nv) : gradKernelOf<ELEM, kLayerNorm, kPostPre>(vector, nv);
  return pass == kPre ? gradKernelOf<ELEM, kRmsNorm, kPre>(vector, nv) : pass == kPost ? gradKernelOf<ELEM, kRmsNorm, kPost>(vector, nv) : gradKernelOf<ELEM, kRmsNorm, kPostPre>(vector, nv);
}
template <int ELEM> GradAheadKernel gradAheadKernel(int kind, int pass, int nv) {
  if (kind == kLayerNorm)
    return pass == kPre ? gradAheadKernelOf<ELEM, kLayerNorm, kPre>(nv) : pass == kPost ? gradAheadKernelOf<ELEM, kLayerNorm, kPost>(nv) : gradAheadKernelOf<ELEM, kLayerNorm, kPostPre>(nv);
  return pass == kPre ? gradAheadKernelOf<ELEM, kRmsNorm, kPre>(nv) : pass == kPost ? gradAheadKernelOf<ELEM, kRmsNorm, kPost>(nv) : gradAheadKernelOf<ELEM, kRmsNorm, kPostPre>(nv);
}

} // namespace kernels
} // namespace afir
