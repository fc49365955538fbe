// Forward row passes: h = normB(x); out = alpha*x + scale*act(gate)*(normA(y)*weight + bias); h = normB(out).
//
// One team of threads per row.  A row is read once and held in registers (f32) across its statistics, so every tensor
// crosses HBM once; the mean and the variance of a layer norm are two sums over those registers, not one sum of
// squares, so that a row far from zero loses nothing.  Statistics, the gate and the sums are f32; `out` and `h` are
// rounded once each, and normB reads `out` as it was rounded, which is what the gradient pass will read.
#pragma once

#include "kernels/loose.cuh"

namespace afir {
namespace kernels {

// Statistics of the row in v (columns at or beyond `cols` are not counted).
template <int KIND, int NV, int VEC>
__device__ __forceinline__ void rowStatistics(Team &team, const float (&v)[NV][VEC], int cols, float eps, float &mean, float &rstd) {
  const float share = 1.0f / static_cast<float>(cols);
  mean = 0.0f;
  if constexpr (KIND == kLayerNorm) {
    float s[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[0] += v[i][e];  // zeros beyond the row
    teamSum(team, s);
    mean = s[0] * share;
  }
  float q[1] = {0.0f};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if ((i * team.lanes + team.lane) * VEC >= cols) continue;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float d = (i * team.lanes + team.lane) * VEC + e < cols ? v[i][e] - mean : 0.0f;
      q[0] += d * d;
    }
  }
  teamSum(team, q);
  rstd = __frsqrt_rn(q[0] * share + eps);
}

template <int ELEM, int KIND, int NV, int VEC>
__device__ __forceinline__ void storeNormed(const Team &team, const float (&v)[NV][VEC], int cols, float mean, float rstd,
                                            const NormVectors &p, int paramType, void *base, int64_t rowAt) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (i * team.lanes + team.lane) * VEC;
    if (col >= cols) continue;
    float w[VEC], r[VEC];
    looseParam<ELEM, VEC>(p.weight, paramType, col, cols, w);
#pragma unroll
    for (int e = 0; e < VEC; ++e) r[e] = (v[i][e] - mean) * rstd * w[e];
    if constexpr (KIND == kLayerNorm) {
      looseParam<ELEM, VEC>(p.bias, paramType, col, cols, w);
#pragma unroll
      for (int e = 0; e < VEC; ++e) r[e] += w[e];
    }
    looseStore<ELEM, VEC>(base, rowAt, col, cols, r);
  }
}

__device__ __forceinline__ void storeStatistics(const Team &team, const NormStatsOut &s, int64_t row, float mean, float rstd) {
  if (team.lane != 0) return;
  if (s.rstd) s.rstd[row] = rstd;
  if (s.mean) s.mean[row] = mean;
}

// Any width and alignment (loose.cuh).  Bound by instructions: the shifts, and the tests at a row's end.  8000 x 4001 bf16 rms
// with a checkpoint 73 us (2.2 TB/s), gated f16 layer 172 us; aligned 8192 x 4096 rows take 66 us here and 37 in
// block_norm_forward_ahead.cuh.
template <int ELEM, int KIND, int PASS, int NV>
__global__ void __launch_bounds__(512) blockNormForwardKernel(const __grid_constant__ BlockNormLaunch p, int teamLanes) {
  gridDependencyPrologue();
  constexpr int VEC = ElemOf<ELEM>::kVec, EB = 16 / VEC;
  __shared__ TeamScratch scratch;
  Team team = makeTeam(teamLanes, scratch);
  const int cols = static_cast<int>(p.cols);
  const int64_t step = static_cast<int64_t>(gridDim.x) * team.count;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * team.count + team.index; row < p.rows; row += step) {
    const RowsIn first = PASS == kPre ? p.x : p.y;
    float v[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * team.lanes + team.lane) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[i][e] = 0.0f;
      if (col < cols) looseLoad<ELEM, VEC>(first.base, row * first.ld, col, cols, innerRow(row, p.rows, first.ld * EB), v[i]);
    }
    if (p.checkpoint.codes) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (i * team.lanes + team.lane) * VEC;
        unsigned int codes[VEC / 4];
        const int e8 = codesOf<ELEM>(pack<ELEM, VEC>(v[i]), codes);  // the values as they were
        if (col >= cols) continue;
        looseCodes(p.checkpoint.codes + row * p.checkpoint.codesLd + col, col, cols, codes);
        if (col % kCheckpointBlock == 0) p.checkpoint.exps[row * p.checkpoint.expsLd + col / kCheckpointBlock] = static_cast<uint8_t>(e8);
      }
    }
    float mean, rstd;
    rowStatistics<KIND, NV, VEC>(team, v, cols, PASS == kPre ? p.epsB : p.epsA, mean, rstd);
    if constexpr (PASS == kPre) {
      storeStatistics(team, p.statsB, row, mean, rstd);
      storeNormed<ELEM, KIND, NV, VEC>(team, v, cols, mean, rstd, p.b, p.paramType, p.h.base, row * p.h.ld);
    } else {
      storeStatistics(team, p.statsA, row, mean, rstd);
      const bool grouped = p.gateForm == kGateGroup;
      const int64_t gateRow = grouped ? row / p.groupRows : row, gateRows = grouped ? (p.rows + p.groupRows - 1) / p.groupRows : p.rows;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (i * team.lanes + team.lane) * VEC;
        if (col >= cols) continue;
        float t[VEC];
        looseParam<ELEM, VEC>(p.a.weight, p.paramType, col, cols, t);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[i][e] = (v[i][e] - mean) * rstd * t[e];
        if constexpr (KIND == kLayerNorm) {
          looseParam<ELEM, VEC>(p.a.bias, p.paramType, col, cols, t);
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[i][e] += t[e];
        }
        if (p.gateForm != kGateNone) {
          looseLoad<ELEM, VEC>(p.gate.base, gateRow * p.gate.ld, col, cols, innerRow(gateRow, gateRows, p.gate.ld * EB), t);
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[i][e] *= gateValue(t[e], p.gateAct);
        }
        if (p.scale) {
          looseParam<ELEM, VEC>(p.scale, p.paramType, col, cols, t);
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[i][e] *= t[e];
        }
        looseLoad<ELEM, VEC>(p.x.base, row * p.x.ld, col, cols, innerRow(row, p.rows, p.x.ld * EB), t);
#pragma unroll
        for (int e = 0; e < VEC; ++e)  // as it is stored
          v[i][e] = ElemOf<ELEM>::widen(ElemOf<ELEM>::narrow(fmaf(p.alpha, t[e], v[i][e])));
        looseStore<ELEM, VEC>(p.out.base, row * p.out.ld, col, cols, v[i]);
      }
      if constexpr (PASS == kPostPre) {
        rowStatistics<KIND, NV, VEC>(team, v, cols, p.epsB, mean, rstd);
        storeStatistics(team, p.statsB, row, mean, rstd);
        storeNormed<ELEM, KIND, NV, VEC>(team, v, cols, mean, rstd, p.b, p.paramType, p.h.base, row * p.h.ld);
      }
    }
  }
}

} // namespace kernels
} // namespace afir
