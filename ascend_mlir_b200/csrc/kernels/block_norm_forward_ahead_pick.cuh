// The instantiations of the forward row kernels that fetch rows ahead, for one element type (one file each).
#pragma once

#include "kernels/block_norm_forward_ahead.cuh"
#include "kernels/block_norm_kernels.h"

namespace afir {
namespace kernels {

template <int ELEM, int KIND, int PASS> ForwardAheadKernel forwardAheadKernelOf(bool full, int nv) {
  if (nv == 1) return full ? blockNormForwardAheadKernel<ELEM, KIND, PASS, true, 1> : blockNormForwardAheadKernel<ELEM, KIND, PASS, false, 1>;
  if (nv == 2) return full ? blockNormForwardAheadKernel<ELEM, KIND, PASS, true, 2> : blockNormForwardAheadKernel<ELEM, KIND, PASS, false, 2>;
  return nullptr;
}
template <int ELEM, int KIND> ForwardAheadKernel forwardAheadKernelOf(int pass, bool full, int nv) {
  if (pass == kPre) return forwardAheadKernelOf<ELEM, KIND, kPre>(full, nv);
  if (pass == kPost) return forwardAheadKernelOf<ELEM, KIND, kPost>(full, nv);
  return forwardAheadKernelOf<ELEM, KIND, kPostPre>(full, nv);
}
template <int ELEM> ForwardAheadKernel forwardAheadKernel(int kind, int pass, bool full, int nv) {
  return kind == kLayerNorm ? forwardAheadKernelOf<ELEM, kLayerNorm>(pass, full, nv) : forwardAheadKernelOf<ELEM, kRmsNorm>(pass, full, nv);
}

} // namespace kernels
} // namespace afir
