#include "kernels/block_norm_grad_pick.cuh"

namespace afir {
namespace kernels {
template GradKernel gradKernel<kF16>(int kind, int pass, int nv);
} // namespace kernels
} // namespace afir
