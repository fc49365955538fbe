#include "kernels/block_norm_forward_pick.cuh"

namespace afir {
namespace kernels {
template ForwardKernel forwardKernel<kF32>(int kind, int pass, bool vector, int nv);
} // namespace kernels
} // namespace afir
