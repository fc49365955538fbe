// Host side of the row passes: which team and kernel a launch takes, how the gradient's rows are split, and the kernel
// that adds the teams' column sums.
#include "kernels/block_norm.h"

#include <algorithm>
#include <mutex>
#include <set>
#include <utility>

#include "kernels/block_norm_kernels.h"
#include "kernels/launch_util.h"

namespace afir {
namespace kernels {
namespace {

// ---- the column sums --------------------------------------------------------------------------------------------
struct FinishParams {
  int layer, elemType, paramType, gateForm, gateAct;
  int64_t cols, groups, chunks, teams, sumsLd;
  const float *sumsA, *sumsB;  // null = that norm is not part of the pass
  const void *weight, *bias, *scale, *gate;
  int64_t gateLd;
  float *dweight, *dbias, *dscale, *nextWeight, *nextBias, *dgate;
  int64_t dgateLd;
};

__device__ __forceinline__ float elemAt(const void *p, int type, int64_t at) {
  if (type == kF32) return static_cast<const float *>(p)[at];
  if (type == kF16) return __half2float(static_cast<const __half *>(p)[at]);
  return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[at]);
}

constexpr int kFinishThreads = 512;

__device__ __forceinline__ float4 plus(const float4 &a, const float4 &b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }

// Four columns per thread.  A warp is QUADS of them (lane % QUADS) by 32 / QUADS slots, a CTA 16 such warps, and slots are
// numbered through the warps.  Adds the slots' values over each run of `slots` neighbouring slots (a power of two): shuffles
// inside a warp, then shared memory across the run's warps.  The first slot of a run gets the sums.
template <int VALUES, int QUADS> __device__ __forceinline__ void slotSums(float4 (&v)[VALUES], float4 (*buf)[kFinishThreads / 32 * QUADS], int slots) {
  constexpr int kPerWarp = 32 / QUADS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < kPerWarp; o *= 2) {
    if (o >= slots) break;
#pragma unroll
    for (int k = 0; k < VALUES; ++k) {
      float4 other;
      other.x = __shfl_xor_sync(0xffffffffu, v[k].x, o * QUADS);
      other.y = __shfl_xor_sync(0xffffffffu, v[k].y, o * QUADS);
      other.z = __shfl_xor_sync(0xffffffffu, v[k].z, o * QUADS);
      other.w = __shfl_xor_sync(0xffffffffu, v[k].w, o * QUADS);
      v[k] = plus(v[k], other);
    }
  }
  if (slots <= kPerWarp) return;
  const int warps = slots / kPerWarp;
  if (lane < QUADS) {
#pragma unroll
    for (int k = 0; k < VALUES; ++k) buf[k][warp * QUADS + lane] = v[k];
  }
  __syncthreads();
  if (lane < QUADS && warp % warps == 0) {
#pragma unroll
    for (int k = 0; k < VALUES; ++k) {
#pragma unroll 4
      for (int w = 1; w < warps; ++w) v[k] = plus(v[k], buf[k][(warp + w) * QUADS + lane]);
    }
  }
  __syncthreads();
}

// The rows of sums first, first + step, ... below `count` (VALUES rows of sumsLd floats each), added.
template <int VALUES>
__device__ __forceinline__ void addRows(const float *sums, int64_t sumsLd, int64_t first, int64_t step, int64_t count, float4 (&v)[VALUES]) {
#pragma unroll
  for (int k = 0; k < VALUES; ++k) v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int64_t r = first; r < count; r += step) {
#pragma unroll
    for (int k = 0; k < VALUES; ++k) v[k] = plus(v[k], *reinterpret_cast<const float4 *>(sums + (r * VALUES + k) * sumsLd));
  }
}

// Slots share the rows of sums; the order in which they are added depends on the sizes alone.  Columns between `cols` and
// sumsLd are read (they are in the workspace) and not stored.  The sums are in L2 (the row kernel has just written them) and
// what counts is how many loads a slot has one behind the other: 148 teams' rows of 8192 columns, two norms, 8.1 us; 592
// teams' of 1024 columns and 8 groups of gates, 13.3 us.
template <int VALUES, int QUADS> __global__ void __launch_bounds__(kFinishThreads) blockNormFinishKernel(const __grid_constant__ FinishParams p) {
  gridDependencyPrologue();
  constexpr int allSlots = kFinishThreads / QUADS;
  __shared__ float4 buf[VALUES][kFinishThreads / 32 * QUADS];
  const int64_t col = (static_cast<int64_t>(blockIdx.x) * QUADS + threadIdx.x % QUADS) * 4;
  const bool live = col < p.cols;
  const int slot = threadIdx.x / QUADS;
  float4 next[VALUES];  // normB's, asked for before normA's are waited for
  if (p.sumsB) addRows<VALUES>(p.sumsB + col, p.sumsLd, slot, allSlots, live ? p.teams : 0, next);
  if (p.sumsA) {
    // slots as (groups at once) x (slots per group)
    int atOnce = 1;
    while (atOnce < p.groups && atOnce < allSlots) atOnce *= 2;
    const int perGroup = allSlots / atOnce;
    float w[4], b[4], scale[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool some = col + j < p.cols;
      w[j] = some ? elemAt(p.weight, p.paramType, col + j) : 0.0f;
      b[j] = some && VALUES > 1 ? elemAt(p.bias, p.paramType, col + j) : 0.0f;
      scale[j] = some && p.scale ? elemAt(p.scale, p.paramType, col + j) : 1.0f;
    }
    float4 total[VALUES];
#pragma unroll
    for (int k = 0; k < VALUES; ++k) total[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int64_t g0 = 0; g0 < p.groups; g0 += atOnce) {
      const int64_t group = g0 + slot / perGroup;
      const bool mine = live && group < p.groups;
      float4 s[VALUES];
      addRows<VALUES>(p.sumsA + group * p.chunks * VALUES * p.sumsLd + col, p.sumsLd, slot & (perGroup - 1), perGroup, mine ? p.chunks : 0, s);
      slotSums<VALUES, QUADS>(s, buf, perGroup);
      if (mine && (slot & (perGroup - 1)) == 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (col + j >= p.cols) break;
          float a = 1.0f;
          const float s0 = reinterpret_cast<const float *>(&s[0])[j], s1 = VALUES > 1 ? reinterpret_cast<const float *>(&s[VALUES - 1])[j] : 0.0f;
          if (p.gateForm == kGateGroup) {
            a = gateValue(elemAt(p.gate, p.elemType, group * p.gateLd + col + j), p.gateAct);
            p.dgate[group * p.dgateLd + col + j] = scale[j] * fmaf(w[j], s0, b[j] * s1) * gateSlope(a, p.gateAct);
          }
          float &t0 = reinterpret_cast<float *>(&total[0])[j];
          t0 = fmaf(a, s0, t0);
          if constexpr (VALUES > 1) {
            float &t1 = reinterpret_cast<float *>(&total[1])[j];
            t1 = fmaf(a, s1, t1);
          }
        }
      }
    }
    if (p.groups > 1) slotSums<VALUES, QUADS>(total, buf, allSlots);
    if (live && slot == 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (col + j >= p.cols) break;
        const float t0 = reinterpret_cast<const float *>(&total[0])[j], t1 = VALUES > 1 ? reinterpret_cast<const float *>(&total[VALUES - 1])[j] : 0.0f;
        p.dweight[col + j] = scale[j] * t0;
        if (p.dbias) p.dbias[col + j] = scale[j] * t1;
        if (p.dscale) p.dscale[col + j] = fmaf(w[j], t0, b[j] * t1);
      }
    }
  }
  if (p.sumsB) {
    slotSums<VALUES, QUADS>(next, buf, allSlots);
    if (live && slot == 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (col + j >= p.cols) break;
        p.nextWeight[col + j] = reinterpret_cast<const float *>(&next[0])[j];
        if (p.nextBias) p.nextBias[col + j] = reinterpret_cast<const float *>(&next[VALUES - 1])[j];
      }
    }
  }
}

// ---- launch shape -----------------------------------------------------------------------------------------------
constexpr size_t kAheadBytes = 225 * 1024;  // of the 227 KB that the CTAs of an SM can have, each with 1 KB of its own

struct TeamShape { int nv, lanes, teamsPerCta; };

TeamShape shapeOf(int vec, int nv, int64_t cols) {
  TeamShape s;
  s.nv = nv;
  const int64_t perThread = static_cast<int64_t>(nv) * vec;
  s.lanes = static_cast<int>(((cols + perThread - 1) / perThread + 31) / 32 * 32);
  s.teamsPerCta = std::max(1, 256 / s.lanes);
  return s;
}

// A CTA per team's row.  One vector per thread while 512 threads are enough, for the shortest way through one row (296 rows of
// 4096 bf16 behind a block: 10.4 us, 12.3 with two); 16 columns per thread where many rows have little to do each: before a
// block (592 rows: 8.2 us, 10.3 with one vector), or in shifted pieces.
TeamShape forwardShape(int elemType, int pass, bool vector, int64_t rows, int64_t cols, int smCount) {
  const int vec = elemType == kF32 ? 4 : 8;
  const int64_t perThread = rows >= 2 * smCount && (pass == kPre || !vector) ? 16 : vec;
  int nv = 1;
  while (nv * vec < perThread && static_cast<int64_t>(nv) * vec * 32 < cols) nv *= 2;
  while (static_cast<int64_t>(nv) * vec * 512 < cols) nv *= 2;
  return shapeOf(vec, nv, cols);
}

// The gradient with rows fetched ahead, 512 threads per SM: two vectors per thread, which share a row's scalars and sums (8192 x
// 4096 f16 rms: 110 us, 136 with one), one of a 16-bit layer norm, whose column sums are twice as many registers (151 us, 712
// with two: they spill), in a team of up to 512 threads; beyond that what the width needs; fewer where that makes every thread's
// vectors lie inside the row, which spares the kernel its tests.
TeamShape gradShape(int elemType, int kind, int64_t cols) {
  const int vec = elemType == kF32 ? 4 : 8;
  int nv = kind == kLayerNorm && elemType != kF32 ? 1 : 2;
  if (nv == 2 && cols % (64 * vec) != 0 && (cols % (32 * vec) == 0 || cols < 32 * vec) && cols <= 512 * vec) nv = 1;
  while (static_cast<int64_t>(nv) * vec * 512 < cols) nv *= 2;
  return shapeOf(vec, nv, cols);
}

GradAheadKernel aheadKernel(int elemType, int kind, int pass, bool token, bool full, int nv) {
  if (kind == kLayerNorm)
    return elemType == kF32   ? gradAheadKernel<kF32, kLayerNorm>(pass, token, full, nv)
           : elemType == kF16 ? gradAheadKernel<kF16, kLayerNorm>(pass, token, full, nv)
                              : gradAheadKernel<kBF16, kLayerNorm>(pass, token, full, nv);
  return elemType == kF32   ? gradAheadKernel<kF32, kRmsNorm>(pass, token, full, nv)
         : elemType == kF16 ? gradAheadKernel<kF16, kRmsNorm>(pass, token, full, nv)
                            : gradAheadKernel<kBF16, kRmsNorm>(pass, token, full, nv);
}

bool rowsAligned(const void *base, int64_t ld, int64_t elemBytes, int64_t bytes) {
  return !base || ((reinterpret_cast<uintptr_t>(base) % static_cast<uintptr_t>(bytes)) == 0 && (ld * elemBytes) % bytes == 0);
}
bool vectorAligned(const void *base) { return (reinterpret_cast<uintptr_t>(base) & 15u) == 0; }

// Columns of the rows that an SM works on at once: what its threads hold, and half of that for f32 rows, of which two
// would not fit in shared memory otherwise.
int64_t gradTeamsPerSm(int elemType, int kind, int64_t cols) {
  const int64_t most = (kind == kLayerNorm ? 4096 : 8192) / (elemType == kF32 ? 2 : 1);
  return std::min<int64_t>(16, std::max<int64_t>(1, most / cols));
}

GradPlan gradPlan(int elemType, int kind, int gateForm, int64_t rows, int64_t cols, int64_t groupRows, int smCount) {
  GradPlan plan = {};
  const int64_t all = std::max<int64_t>(rows, 1);
  const int64_t perGroup = gateForm == kGateGroup ? std::min(groupRows, all) : all;
  const int64_t groups = gateForm == kGateGroup ? (rows + perGroup - 1) / perGroup : 1;
  // As many teams as an SM holds: enough rows under way to cover a row's two sums, few enough that the teams' sums (f32, one
  // or two rows each) stay small beside the rows.
  const int64_t teams = std::max<int64_t>(1, std::min<int64_t>(rows, smCount * gradTeamsPerSm(elemType, kind, cols)));
  const int64_t wanted = std::max<int64_t>(1, groups ? teams / groups : 1);
  const int64_t chunkRows = (perGroup + wanted - 1) / wanted;
  const int64_t chunks = (perGroup + chunkRows - 1) / chunkRows;
  plan.groups = static_cast<int>(groups);
  plan.groupRows = static_cast<int>(perGroup);
  plan.chunkRows = static_cast<int>(chunkRows);
  plan.chunks = static_cast<int>(chunks);
  plan.teams = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(teams, groups * chunks)));
  plan.sumsLd = static_cast<int>((cols + 3) / 4 * 4);
  return plan;
}

int64_t sumsFloats(const GradPlan &plan, int pass, int kind) {
  const int64_t values = kind == kLayerNorm ? 2 : 1;
  return values * plan.sumsLd * ((pass != kPre ? static_cast<int64_t>(plan.groups) * plan.chunks : 0) + (pass != kPost ? plan.teams : 0));
}

} // namespace

cudaError_t reserveSharedMemory(const void *kernel, int bytes) {
  static std::mutex mu;
  static std::set<std::pair<const void *, int>> done;
  int device = 0;
  if (const cudaError_t e = cudaGetDevice(&device); e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lock(mu);
  if (done.count({kernel, device})) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.insert({kernel, device});
  return e;
}

int launchBlockNorm(const BlockNormLaunch &l, cudaStream_t stream, int *launched) {
  if (launched) *launched = 0;
  if (l.rows == 0) return 0;
  if (l.cols <= 0 || l.cols > kMaxNormCols || l.rows > kMaxNormRows) return cudaErrorInvalidValue;
  const int64_t eb = elemBytes(l.elemType);
  const int vec = static_cast<int>(16 / eb);
  bool vector = l.cols % vec == 0;
  for (const RowsIn &r : {l.x, l.y, l.gate}) vector = vector && rowsAligned(r.base, r.ld, eb, 16);
  for (const RowsOut &r : {l.out, l.h}) vector = vector && rowsAligned(r.base, r.ld, eb, 16);
  for (const void *v : {l.a.weight, l.a.bias, l.b.weight, l.b.bias, l.scale}) vector = vector && vectorAligned(v);
  vector = vector && rowsAligned(l.checkpoint.codes, l.checkpoint.codesLd, 1, vec);
  int device = 0;
  if (const cudaError_t e = cudaGetDevice(&device); e != cudaSuccess) return e;
  const int sms = deviceSmCount(device);
  // Rows fetched ahead by teams that stay, where every team gets two rows or more and two fit in shared memory beside the
  // parameters: 1024 threads per SM (64 registers each) before a block, up to 768 (80 registers) behind it, in one CTA that
  // shares its parameters.  Two rows each (888 x 4096 f16 layer, behind a block): 20.5 us, 24.6 without; eight: 41 and 67; before
  // a block, 4096 bf16 rms, two, four and sixteen: 11.2, 18.4 and 41 us, 12.3, 20.5 and 55 without; one row each gains nothing,
  // and few teams' set-up costs 2 us.
  if (vector) {
    TeamShape s = gradShape(l.elemType, kRmsNorm, l.cols);
    if (s.nv <= 2) {
      const int ctaThreads = l.pass == kPre ? kForwardAheadThreads : kForwardAheadPostThreads, ctasPerSm = l.pass == kPre ? 2 : 1;
      s.teamsPerCta = std::max(1, std::min(15, ctaThreads / s.lanes));
      const int threads = s.lanes * s.teamsPerCta;
      const int tensors = l.pass == kPre ? 1 : l.gateForm != kGateNone ? 3 : 2;
      const int vectors = (l.kind == kLayerNorm ? 2 : 1) * (l.pass == kPostPre ? 2 : 1);
      const size_t paramBytes = static_cast<size_t>(vectors) * static_cast<size_t>(s.lanes * s.nv * vec) * sizeof(float);
      const size_t rowBytes = static_cast<size_t>(tensors) * static_cast<size_t>(s.nv) * 16 * static_cast<size_t>(ctaThreads);
      const size_t perCta = kAheadBytes / static_cast<size_t>(ctasPerSm) - 1536;
      const int stages = static_cast<int>(std::min<size_t>(4, (perCta - std::min(perCta, paramBytes)) / rowBytes));
      if (stages >= 2 && l.rows >= static_cast<int64_t>(2) * sms * ctasPerSm * s.teamsPerCta) {
        const bool full = static_cast<int64_t>(s.lanes) * s.nv * vec == l.cols;
        const ForwardAheadKernel kernel = l.elemType == kF32   ? forwardAheadKernel<kF32>(l.kind, l.pass, full, s.nv)
                                          : l.elemType == kF16 ? forwardAheadKernel<kF16>(l.kind, l.pass, full, s.nv)
                                                               : forwardAheadKernel<kBF16>(l.kind, l.pass, full, s.nv);
        cudaError_t e = reserveSharedMemory(reinterpret_cast<const void *>(kernel), static_cast<int>(kAheadBytes));
        if (e != cudaSuccess) return e;
        e = launchDependent(kernel, dim3(static_cast<unsigned int>(sms * ctasPerSm)), dim3(static_cast<unsigned int>(threads)),
                            static_cast<size_t>(stages) * rowBytes + paramBytes, stream, l, s.lanes, stages);
        if (e == cudaSuccess && launched) *launched += 1;
        return e;
      }
    }
  }
  const TeamShape s = forwardShape(l.elemType, l.pass, vector, l.rows, l.cols, sms);
  const ForwardKernel kernel = l.elemType == kF32   ? forwardKernel<kF32>(l.kind, l.pass, vector, s.nv)
                               : l.elemType == kF16 ? forwardKernel<kF16>(l.kind, l.pass, vector, s.nv)
                                                    : forwardKernel<kBF16>(l.kind, l.pass, vector, s.nv);
  if (!kernel) return cudaErrorInvalidValue;
  const int64_t ctas = (l.rows + s.teamsPerCta - 1) / s.teamsPerCta;
  const unsigned int grid = static_cast<unsigned int>(std::min<int64_t>(ctas, 0x7fffffff));
  const cudaError_t e = launchDependent(kernel, dim3(grid), dim3(static_cast<unsigned int>(s.lanes * s.teamsPerCta)), 0, stream, l, s.lanes);
  if (e == cudaSuccess && launched) *launched += 1;
  return e;
}

size_t blockNormGradWorkspaceBytes(int pass, int elemType, int kind, int gateForm, int64_t rows, int64_t cols, int64_t groupRows, int smCount) {
  return static_cast<size_t>(sumsFloats(gradPlan(elemType, kind, gateForm, rows, cols, groupRows, smCount), pass, kind)) * sizeof(float);
}

int launchBlockNormGrad(const BlockNormGradLaunch &l, cudaStream_t stream, int *launched) {
  if (launched) *launched = 0;
  if (l.cols <= 0 || l.cols > kMaxNormCols || l.rows > kMaxNormRows) return cudaErrorInvalidValue;
  int device = 0;
  if (const cudaError_t e = cudaGetDevice(&device); e != cudaSuccess) return e;
  const int sms = deviceSmCount(device);
  GradPlan plan = gradPlan(l.elemType, l.kind, l.gateForm, l.rows, l.cols, l.groupRows, sms);
  const size_t need = static_cast<size_t>(sumsFloats(plan, l.pass, l.kind)) * sizeof(float);
  if (!l.workspace || l.workspaceBytes < need || !vectorAligned(l.workspace)) return cudaErrorInvalidValue;
  const int64_t values = l.kind == kLayerNorm ? 2 : 1;
  if (l.pass != kPre) plan.sumsA = static_cast<float *>(l.workspace);
  if (l.pass != kPost) plan.sumsB = static_cast<float *>(l.workspace) + (l.pass != kPre ? static_cast<int64_t>(plan.groups) * plan.chunks * values * plan.sumsLd : 0);

  if (l.rows > 0) {
    const int64_t eb = elemBytes(l.elemType);
    const int vec = static_cast<int>(16 / eb);
    bool vector = l.cols % vec == 0;
    for (const RowsIn &r : {l.dout, l.dh, l.source, l.y, l.gate}) vector = vector && rowsAligned(r.base, r.ld, eb, 16);
    for (const RowsOut &r : {l.dx, l.dy}) vector = vector && rowsAligned(r.base, r.ld, eb, 16);
    if (l.gateForm == kGateToken) vector = vector && rowsAligned(l.dgate.base, l.dgate.ld, eb, 16);
    for (const void *v : {l.a.weight, l.a.bias, l.b.weight, l.scale}) vector = vector && vectorAligned(v);
    vector = vector && rowsAligned(l.checkpoint.codes, l.checkpoint.codesLd, 1, vec);
    TeamShape s = gradShape(l.elemType, l.kind, l.cols);
    // (few teams: spread over the SMs)
    s.teamsPerCta = std::max(1, std::min({15, kGradAheadThreads / s.lanes, (plan.teams + sms - 1) / sms}));
    // rows fetched ahead: as many (2 to 4) as a CTA has shared memory for beside its parameters; rows too wide for two take
    // the kernel without
    const int tensors = (l.pass != kPost ? 2 : 0) + (l.dout.base ? 1 : 0) + (l.pass != kPre ? 1 : 0) + (l.gateForm == kGateToken ? 1 : 0);
    const int vectors = (l.pass != kPost ? 1 : 0) + (l.pass != kPre ? 1 : 0) + (l.gateForm == kGateToken && l.kind == kLayerNorm ? 1 : 0);
    const size_t paramBytes = static_cast<size_t>(vectors) * static_cast<size_t>(s.nv * vec) * kGradAheadThreads * sizeof(float);
    const size_t rowBytes = static_cast<size_t>(tensors) * static_cast<size_t>(s.nv) * 16 * kGradAheadThreads;
    const size_t perCta = kAheadBytes - 1536;
    const int stages = static_cast<int>(std::min<size_t>(4, std::max<size_t>(2, (perCta - std::min(perCta, paramBytes)) / rowBytes)));
    const size_t slotBytes = static_cast<size_t>(stages) * rowBytes + paramBytes;
    const GradAheadKernel ahead = vector && slotBytes <= kAheadBytes ? aheadKernel(l.elemType, l.kind, l.pass, l.gateForm == kGateToken, static_cast<int64_t>(s.lanes) * s.nv * vec == l.cols, s.nv) : nullptr;
    const unsigned int threads = static_cast<unsigned int>(s.lanes * s.teamsPerCta);
    const dim3 grid(static_cast<unsigned int>((plan.teams + s.teamsPerCta - 1) / s.teamsPerCta));
    cudaError_t e;
    if (ahead) {
      if (e = reserveSharedMemory(reinterpret_cast<const void *>(ahead), static_cast<int>(kAheadBytes)); e != cudaSuccess) return e;
      e = launchDependent(ahead, grid, dim3(threads), slotBytes, stream, l, plan, s.lanes, stages);
    } else {
      const GradKernel kernel = l.elemType == kF32   ? gradKernel<kF32>(l.kind, l.pass, s.nv)
                                : l.elemType == kF16 ? gradKernel<kF16>(l.kind, l.pass, s.nv)
                                                     : gradKernel<kBF16>(l.kind, l.pass, s.nv);
      if (!kernel) return cudaErrorInvalidValue;
      e = launchDependent(kernel, grid, dim3(threads), 0, stream, l, plan, s.lanes);
    }
    if (e != cudaSuccess) return e;
    if (launched) *launched += 1;
  }
  FinishParams f = {};
  f.layer = l.kind == kLayerNorm;
  f.elemType = l.elemType;
  f.paramType = l.paramType;
  f.gateForm = l.gateForm;
  f.gateAct = l.gateAct;
  f.cols = l.cols;
  f.sumsLd = plan.sumsLd;
  f.groups = plan.groups;
  f.chunks = l.rows > 0 ? plan.chunks : 0;  // no rows: the gradients are sums of nothing
  f.teams = l.rows > 0 ? plan.teams : 0;
  f.sumsA = l.pass != kPre ? plan.sumsA : nullptr;
  f.sumsB = l.pass != kPost ? plan.sumsB : nullptr;
  f.weight = l.a.weight;
  f.bias = l.a.bias;
  f.scale = l.scale;
  f.gate = l.gate.base;
  f.gateLd = l.gate.ld;
  f.dweight = l.da.weight;
  f.dbias = l.da.bias;
  f.dscale = l.dscale;
  f.nextWeight = l.db.weight;
  f.nextBias = l.db.bias;
  f.dgate = static_cast<float *>(l.gateForm == kGateGroup ? l.dgate.base : nullptr);
  f.dgateLd = l.dgate.ld;
  // whole 128-byte lines of the sums (8 threads of 4 columns) for wide rows, half lines, twice the slots and CTAs else (whole
  // gradient, 8192 columns: 186 us, 189 with half lines; 1024 columns: 36 us, 40 with whole ones)
  const int quads = l.cols >= 4096 ? 8 : 4;
  const unsigned int grid = static_cast<unsigned int>((l.cols + 4 * quads - 1) / (4 * quads));
  const auto finish = f.layer ? (quads == 8 ? blockNormFinishKernel<2, 8> : blockNormFinishKernel<2, 4>)
                              : (quads == 8 ? blockNormFinishKernel<1, 8> : blockNormFinishKernel<1, 4>);
  const cudaError_t e = launchDependent(finish, dim3(grid), dim3(kFinishThreads), 0, stream, f);
  if (e == cudaSuccess && launched) *launched += 1;
  return e;
}

} // namespace kernels
} // namespace afir
