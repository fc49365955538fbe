// Which instantiation of the row kernels a launch takes; one translation unit per element type and direction.
#pragma once

#include "kernels/block_norm.h"
#include "kernels/block_norm_grad.cuh"

namespace afir {
namespace kernels {

// `vector`: everything is aligned for 16-byte accesses; nv = vectors per thread.
using ForwardKernel = void (*)(const BlockNormLaunch, int);
using GradKernel = void (*)(const BlockNormGradLaunch, const GradPlan, int);
template <int ELEM> ForwardKernel forwardKernel(int kind, int pass, bool vector, int nv);
// Teams that stay, with rows fetched ahead (block_norm_forward_ahead.cuh).
using ForwardAheadKernel = void (*)(const BlockNormLaunch, int, int);
template <int ELEM> ForwardAheadKernel forwardAheadKernel(int kind, int pass, bool full, int nv);
template <int ELEM> GradKernel gradKernel(int kind, int pass, int nv);
// With rows fetched ahead (block_norm_grad_vector.cuh); null where a thread would hold more than it has registers for.
using GradAheadKernel = void (*)(const BlockNormGradLaunch, const GradPlan, int, int);
template <int ELEM, int KIND> GradAheadKernel gradAheadKernel(int pass, bool token, bool full, int nv);

} // namespace kernels
} // namespace afir
