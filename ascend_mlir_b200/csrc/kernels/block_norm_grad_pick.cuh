// The instantiations of the gradient row kernels for one element type (included by one file per type).
#pragma once

#include "kernels/block_norm_grad.cuh"
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
template <int ELEM> GradKernel gradKernel(int kind, int pass, bool vector, int nv) {
  if (kind == kLayerNorm)
    return pass == kPre ? gradKernelOf<ELEM, kLayerNorm, kPre>(vector, nv) : pass == kPost ? gradKernelOf<ELEM, kLayerNorm, kPost>(vector, nv) : gradKernelOf<ELEM, kLayerNorm, kPostPre>(vector, nv);
  return pass == kPre ? gradKernelOf<ELEM, kRmsNorm, kPre>(vector, nv) : pass == kPost ? gradKernelOf<ELEM, kRmsNorm, kPost>(vector, nv) : gradKernelOf<ELEM, kRmsNorm, kPostPre>(vector, nv);
}
} // namespace kernels
} // namespace afir
