// 8-bit activation checkpoints: pack (x -> codes and exponents) and restore (-> values in the type again).
//
// value = e4m3(code) * 2^(exp - 127), one power of two per row and 128 columns: the restored value is exact in the type
// the tensor had, so what a checkpoint loses is the one rounding to four significant bits.  1 + 1/128 bytes per element
// for 2 or 4.  Both are one pass over the data, bound by HBM: 16384 x 8192 bf16 packed in 74 us (403 MB, 5.4 TB/s: 83 % of a
// plain copy's rate); rows of odd widths by instructions, 8000 x 4001 bf16 in 33 us.
#include "kernels/block_norm.h"

#include <algorithm>

#include "kernels/launch_util.h"
#include "kernels/loose.cuh"

namespace afir {
namespace kernels {
namespace {

constexpr int kThreads = 256;

// 128 columns are 16 lanes (8 columns each, 16-bit types) or 32 lanes (4 each, f32).  A team of whole warps walks a row,
// kAhead vectors per thread at a time, all loaded before the first is used; a row may end inside a block.  LOOSE: rows of any
// width and alignment (loose.cuh).
constexpr int kAhead = 4;
template <int ELEM, bool LOOSE>
__global__ void __launch_bounds__(kThreads) checkpointPackKernel(const __grid_constant__ CheckpointPackLaunch p, int lanes) {
  gridDependencyPrologue();
  constexpr int VEC = ElemOf<ELEM>::kVec;
  const int cols = static_cast<int>(p.cols);
  const int teams = kThreads / lanes, team = static_cast<int>(threadIdx.x) / lanes, lane = static_cast<int>(threadIdx.x) - team * lanes;
  const int64_t step = static_cast<int64_t>(gridDim.x) * teams;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * teams + team; row < p.rows; row += step) {
    const char *from = static_cast<const char *>(p.x.base) + row * p.x.ld * (16 / VEC);
    for (int base = lane * VEC; base - lane * VEC < cols; base += lanes * VEC * kAhead) {
      uint4 raw[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int col = base + i * lanes * VEC;
        if constexpr (LOOSE) {
          float v[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[e] = 0.0f;
          if (col < cols) looseLoad<ELEM, VEC>(p.x.base, row * p.x.ld, col, cols, innerRow(row, p.rows, p.x.ld * (16 / VEC)), v);
          raw[i] = pack<ELEM, VEC>(v);  // the values as they were
        } else raw[i] = col < cols ? *reinterpret_cast<const uint4 *>(from + static_cast<int64_t>(col) * (16 / VEC)) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int col = base + i * lanes * VEC;
        if (col - lane * VEC >= cols) break;  // the whole team's
        if constexpr (LOOSE) {
          unsigned int codes[VEC / 4];
          const int e8 = codesOf<ELEM>(raw[i], codes);
          if (col >= cols) continue;
          looseCodes(p.out.codes + row * p.out.codesLd + col, col, cols, codes);
          if (col % kCheckpointBlock == 0) p.out.exps[row * p.out.expsLd + col / kCheckpointBlock] = static_cast<uint8_t>(e8);
        } else packVector<ELEM>(raw[i], col < cols, col, row, p.out);
      }
    }
  }
}

template <int ELEM, bool LOOSE>
__global__ void __launch_bounds__(kThreads) checkpointRestoreKernel(const __grid_constant__ CheckpointRestoreLaunch p) {
  gridDependencyPrologue();
  constexpr int VEC = ElemOf<ELEM>::kVec;
  const int cols = static_cast<int>(p.cols);
  const int64_t perRow = (p.cols + VEC - 1) / VEC;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; u < p.rows * perRow; u += step) {
    const int64_t row = u / perRow;
    const int col = static_cast<int>(u - row * perRow) * VEC;
    if constexpr (LOOSE) {
      float v[VEC];
      looseCheckpoint<VEC>(p.in, row, col, cols, innerRow(row, p.rows, p.in.codesLd), v);
      looseStore<ELEM, VEC>(p.out.base, row * p.out.ld, col, cols, v);
    } else {
      const uint8_t *from = p.in.codes + row * p.in.codesLd + col;
      F2 v[VEC / 2];
      const uint2 codes = VEC == 8 ? *reinterpret_cast<const uint2 *>(from) : make_uint2(*reinterpret_cast<const unsigned int *>(from), 0u);
      codePairs<ELEM>(codes, p.in.exps[row * p.in.expsLd + col / kCheckpointBlock], v);
      storePairs<ELEM>(p.out.base, row * p.out.ld + col, v);
    }
  }
}

bool aligned(const void *base, int64_t rowBytes, int64_t bytes) {
  return (reinterpret_cast<uintptr_t>(base) % static_cast<uintptr_t>(bytes)) == 0 && rowBytes % bytes == 0;
}
unsigned int gridFor(int64_t units, int64_t perCta) {
  int device = 0;
  cudaGetDevice(&device);
  const int64_t ctas = (units + perCta - 1) / perCta;
  return static_cast<unsigned int>(std::max<int64_t>(1, std::min<int64_t>(ctas, static_cast<int64_t>(deviceSmCount(device)) * 64)));
}

} // namespace

int launchCheckpointPack(const CheckpointPackLaunch &l, cudaStream_t stream, int *launched) {
  if (l.rows == 0) return 0;
  if (l.cols <= 0 || l.cols > (1ll << 30)) return cudaErrorInvalidValue;
  const int64_t eb = elemBytes(l.elemType), vec = 16 / eb;
  const bool vector = l.cols % vec == 0 && aligned(l.x.base, l.x.ld * eb, 16) && aligned(l.out.codes, l.out.codesLd, vec);
  const auto kernel = l.elemType == kF32   ? (vector ? checkpointPackKernel<kF32, false> : checkpointPackKernel<kF32, true>)
                      : l.elemType == kF16 ? (vector ? checkpointPackKernel<kF16, false> : checkpointPackKernel<kF16, true>)
                                           : (vector ? checkpointPackKernel<kBF16, false> : checkpointPackKernel<kBF16, true>);
  int lanes = 32;  // the fewest (32, 64, 128 or 256) that take a row at one go
  while (lanes < kThreads && lanes * vec * kAhead < l.cols) lanes *= 2;
  const cudaError_t e = launchDependent(kernel, dim3(gridFor(l.rows, kThreads / lanes)), dim3(kThreads), 0, stream, l, lanes);
  if (e == cudaSuccess && launched) *launched += 1;
  return e;
}

int launchCheckpointRestore(const CheckpointRestoreLaunch &l, cudaStream_t stream, int *launched) {
  if (l.rows == 0) return 0;
  if (l.cols <= 0 || l.cols > (1ll << 30)) return cudaErrorInvalidValue;
  const int64_t eb = elemBytes(l.elemType), vec = 16 / eb;
  const bool vector = l.cols % vec == 0 && aligned(l.out.base, l.out.ld * eb, 16) && aligned(l.in.codes, l.in.codesLd, vec);
  const auto kernel = l.elemType == kF32   ? (vector ? checkpointRestoreKernel<kF32, false> : checkpointRestoreKernel<kF32, true>)
                      : l.elemType == kF16 ? (vector ? checkpointRestoreKernel<kF16, false> : checkpointRestoreKernel<kF16, true>)
                                           : (vector ? checkpointRestoreKernel<kBF16, false> : checkpointRestoreKernel<kBF16, true>);
  const cudaError_t e = launchDependent(kernel, dim3(gridFor(l.rows * ((l.cols + vec - 1) / vec), kThreads)), dim3(kThreads), 0, stream, l);
  if (e == cudaSuccess && launched) *launched += 1;
  return e;
}

} // namespace kernels
} // namespace afir
