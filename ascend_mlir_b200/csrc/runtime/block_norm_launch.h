// Launches of the operator classes (block_norm, checkpoint, checkpoint_grad): argument roles resolved against concrete
// sizes, checked, and handed to the kernels of kernels/block_norm.h.
#pragma once

#include "runtime/launcher.h"

namespace afir {

inline bool isOperatorClass(KernelClass c) {
  return c == KernelClass::BlockNorm || c == KernelClass::Checkpoint || c == KernelClass::CheckpointGrad;
}
Status operatorWorkspaceBytes(const LaunchDescriptor &d, const std::map<std::string, int64_t> &tiling, int device, size_t &bytes);
Status launchOperator(const LaunchDescriptor &d, const std::map<std::string, int64_t> &tiling, const LaunchArgs &args, LaunchInfo &info);

} // namespace afir
