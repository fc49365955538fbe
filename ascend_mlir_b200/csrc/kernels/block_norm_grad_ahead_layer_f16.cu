#include "kernels/block_norm_grad_ahead_pick.cuh"

namespace afir {
namespace kernels {
template GradAheadKernel gradAheadKernel<kF16, kLayerNorm>(int pass, bool token, bool full, int nv);
} // namespace kernels
} // namespace afir
