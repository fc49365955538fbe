// Which instantiation of the row kernels a launch takes; one translation unit per element type and direction.
#pragma once

#include "kernels/block_norm.h"
#include "kernels/block_norm_grad.cuh"

namespace afir {
namespace kernels {

// VEC = 16-byte accesses; NV = vectors (or, without them, elements) per thread.
constexpr int kScalarSmall = 8, kScalarLarge = 32;

using ForwardKernel = void (*)(const BlockNormLaunch, int);
using GradKernel = void (*)(const BlockNormGradLaunch, const GradPlan, int);
template <int ELEM> ForwardKernel forwardKernel(int kind, int pass, bool vector, int nv);
template <int ELEM> GradKernel gradKernel(int kind, int pass, bool vector, int nv);

} // namespace kernels
} // namespace afir
