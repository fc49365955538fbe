// The instantiations of the gradient row kernels that fetch rows ahead, for one element type and norm (one file each).
#pragma once

#include "kernels/block_norm_grad_vector.cuh"
#include "kernels/block_norm_kernels.h"

namespace afir {
namespace kernels {

template <int ELEM, int KIND, int PASS, bool TOKEN, bool FULL> GradAheadKernel gradAheadKernelOf(int nv) {
  switch (nv) {
  case 1: return blockNormGradVectorKernel<ELEM, KIND, PASS, TOKEN, FULL, 1>;
  case 2: return blockNormGradVectorKernel<ELEM, KIND, PASS, TOKEN, FULL, 2>;
  default: return nullptr;
  }
}
template <int ELEM, int KIND, int PASS, bool TOKEN> GradAheadKernel gradAheadKernelOf(bool full, int nv) {
  return full ? gradAheadKernelOf<ELEM, KIND, PASS, TOKEN, true>(nv) : gradAheadKernelOf<ELEM, KIND, PASS, TOKEN, false>(nv);
}
template <int ELEM, int KIND> GradAheadKernel gradAheadKernel(int pass, bool token, bool full, int nv) {
  if (pass == kPre) return gradAheadKernelOf<ELEM, KIND, kPre, false>(full, nv);
  if (pass == kPost) return token ? gradAheadKernelOf<ELEM, KIND, kPost, true>(full, nv) : gradAheadKernelOf<ELEM, KIND, kPost, false>(full, nv);
  return token ? gradAheadKernelOf<ELEM, KIND, kPostPre, true>(full, nv) : gradAheadKernelOf<ELEM, KIND, kPostPre, false>(full, nv);
}

} // namespace kernels
} // namespace afir
