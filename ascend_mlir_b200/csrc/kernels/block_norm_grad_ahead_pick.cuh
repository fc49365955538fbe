// The instantiations of the gradient row kernels that fetch rows ahead, for one element type and norm (one file each).
#pragma once

#include "kernels/block_norm_grad_vector.cuh"
#include "kernels/block_norm_kernels.h"

namespace afir {
namespace kernels {

template <int ELEM, int KIND, int PASS, int GATE> GradAheadKernel gradAheadKernelOf(int nv) {
  switch (nv) {
  case 1: return blockNormGradVectorKernel<ELEM, KIND, PASS, GATE, 1>;
  case 2: return blockNormGradVectorKernel<ELEM, KIND, PASS, GATE, 2>;
  case 4:
    if constexpr (ELEM == kF32) return blockNormGradVectorKernel<ELEM, KIND, PASS, GATE, 4>;
    else return nullptr;
  default: return nullptr;
  }
}
template <int ELEM, int KIND, int PASS> GradAheadKernel gradAheadKernelOf(int gate, int nv) {
  if (gate == kGateToken) return gradAheadKernelOf<ELEM, KIND, PASS, kGateToken>(nv);
  if (gate == kGateGroup) return gradAheadKernelOf<ELEM, KIND, PASS, kGateGroup>(nv);
  return gradAheadKernelOf<ELEM, KIND, PASS, kGateNone>(nv);
}
template <int ELEM, int KIND> GradAheadKernel gradAheadKernel(int pass, int gate, int nv) {
  if (pass == kPre) return gradAheadKernelOf<ELEM, KIND, kPre, kGateNone>(nv);
  return pass == kPost ? gradAheadKernelOf<ELEM, KIND, kPost>(gate, nv) : gradAheadKernelOf<ELEM, KIND, kPostPre>(gate, nv);
}

} // namespace kernels
} // namespace afir
