#include "kernels/block_norm_forward_ahead_pick.cuh"

namespace afir {
namespace kernels {
template ForwardAheadKernel forwardAheadKernel<kF32>(int kind, int pass, bool full, int nv);
} // namespace kernels
} // namespace afir
