// Launch interface of the row passes around a residual block and of 8-bit activation checkpoints: norms, the gated
// residual sum, their gradients, and the weight gradient that reads a checkpoint.  Plain structs, filled in by the
// runtime (.cpp) and turned into launches by the .cu files.
//
// A residual block:   h = normB(x);  y = block(h);  out = alpha*x + scale * act(gate) * (normA(y)*weight + bias)
// and the next block begins with  h = normB(out).  One kernel family covers the three passes:
//   kPre      h   = normB(x)                                      (before the first block)
//   kPost     out = alpha*x + scale*act(gate)*normA(y)            (after the last one)
//   kPostPre  both: `out` and the next block's h, `out` read by normB as it is stored
#pragma once

#include <cstddef>
#include <cstdint>

#include "kernels/kernels.h"

namespace afir {
namespace kernels {

constexpr int64_t kMaxNormCols = 16384;  // a row stays in the registers of one team of at most 512 threads
constexpr int64_t kMaxNormRows = 1ll << 30;  // rows, and rows of column sums, are counted in 32 bits
constexpr int kCheckpointBlock = 128;    // columns that share one power of two

// Threads of a CTA (at most) in the kernels that fetch rows ahead; a row's slots are laid out for that many.
constexpr int kForwardAheadThreads = 512, kForwardAheadPostThreads = 768, kGradAheadThreads = 512;

enum NormPass : int { kPre = 0, kPost = 1, kPostPre = 2 };
enum NormKind : int { kRmsNorm = 0, kLayerNorm = 1 };
enum GateForm : int { kGateNone = 0, kGateToken = 1, kGateGroup = 2 };  // none; a value per element; a row per group of rows
enum GateAct : int { kActNone = 0, kActSigmoid = 1, kActTanh = 2 };

// Rows of a [rows, cols] tensor: `ld` elements from one row to the next.
struct RowsIn { const void *base; int64_t ld; };
struct RowsOut { void *base; int64_t ld; };

// An activation in 8 bits: e4m3 codes [rows, cols] and, per row and 128 columns, the biased exponent of the power of two
// that the code is multiplied by: value = e4m3(code) * 2^(exp - 127), exact in the type it was made from.
struct CheckpointIn { const uint8_t *codes; int64_t codesLd; const uint8_t *exps; int64_t expsLd; };
struct CheckpointOut { uint8_t *codes; int64_t codesLd; uint8_t *exps; int64_t expsLd; };

struct NormVectors { const void *weight, *bias; };      // [cols], paramType; bias null for an rms norm
struct NormStatsIn { const float *rstd, *mean; };       // [rows]; mean null for an rms norm
struct NormStatsOut { float *rstd, *mean; };            // null = not wanted
struct NormSums { float *weight, *bias; };              // gradients of NormVectors, [cols]

struct BlockNormLaunch {
  int pass, kind, elemType, paramType;
  int64_t rows, cols;
  RowsIn x, y;                 // y: kPost, kPostPre
  NormVectors a, b;            // a: norm of y; b: norm of the stream
  int gateForm, gateAct;
  RowsIn gate;
  int64_t groupRows;           // rows that share a gate row (kGateGroup), at most `rows`
  const void *scale;           // [cols] or null
  float alpha, epsA, epsB;
  RowsOut out, h;
  NormStatsOut statsA, statsB;
  CheckpointOut checkpoint;    // of the tensor normed first: y (kPost, kPostPre) or x; codes null = none
};
int launchBlockNorm(const BlockNormLaunch &l, cudaStream_t stream, int *launched);

struct BlockNormGradLaunch {
  int pass, kind, elemType, paramType;
  int64_t rows, cols;
  RowsIn dout;                 // gradient of the stream behind the block, or null (kPre: of x's other uses)
  RowsIn dh;                   // kPre, kPostPre
  RowsIn source;               // what normB read: x (kPre) or out (kPostPre)
  RowsIn y;                    // kPost, kPostPre
  CheckpointIn checkpoint;     // in the place of the tensor normed first (`source` for kPre, else `y`); codes null = none
  NormVectors a, b;
  NormStatsIn statsA, statsB;
  int gateForm, gateAct;
  RowsIn gate;
  int64_t groupRows;
  const void *scale;
  float alpha;
  RowsOut dx, dy;
  RowsOut dgate;               // kGateToken: elemType; kGateGroup: f32 [groups, cols]
  NormSums da, db;
  float *dscale;
  void *workspace;
  size_t workspaceBytes;
};
size_t blockNormGradWorkspaceBytes(int pass, int elemType, int kind, int gateForm, int64_t rows, int64_t cols, int64_t groupRows, int smCount);
int launchBlockNormGrad(const BlockNormGradLaunch &l, cudaStream_t stream, int *launched);

struct CheckpointPackLaunch {
  int elemType;
  int64_t rows, cols;
  RowsIn x;
  CheckpointOut out;
};
int launchCheckpointPack(const CheckpointPackLaunch &l, cudaStream_t stream, int *launched);

struct CheckpointRestoreLaunch {
  int elemType;
  int64_t rows, cols;
  CheckpointIn in;
  RowsOut out;
};
int launchCheckpointRestore(const CheckpointRestoreLaunch &l, cudaStream_t stream, int *launched);

// dweight[cols, outCols] = restore(in)[rows, cols]^T . dy[rows, outCols]  (checkpoint_grad_tcgen05.cu)
struct CheckpointGradLaunch {
  int elemType;                // of dy, and what the checkpoint was made from: kF16 or kBF16
  int outType;                 // elemType or kF32
  int64_t rows, cols, outCols;
  CheckpointIn in;
  RowsIn dy;
  RowsOut out;
  int accumulate;              // add to what `out` (f32) holds
  int statusWord;              // which of the device's words takes a pipeline wait that ran out
  void *workspace;
  size_t workspaceBytes;
};
size_t checkpointGradWorkspaceBytes(int64_t cols, int64_t outCols, int64_t rows, int smCount);
int launchCheckpointGrad(const CheckpointGradLaunch &l, cudaStream_t stream, int *launched, char *errorText);

// Words that the weight gradient reports a wait that ran out in.  They are part of the library on each device, so a launch
// needs no memory for its word, and a graph that is replayed late writes into one that is still there.
constexpr int kCheckpointGradStatusWords = 4096;
// Reads one of the current device's words, and clears it.  0: no wait ran out; else the error in errorText (256 bytes).
int checkpointGradCheckStatus(int word, char *errorText);

} // namespace kernels
} // namespace afir
