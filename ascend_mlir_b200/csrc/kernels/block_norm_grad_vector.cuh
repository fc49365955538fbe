// The gradient row kernel for rows in 16-byte vectors (formulas and the split of the rows: block_norm_grad.cuh).
//
// A row of the longest form is five tensors in and three out, so a team that loads when it needs the data leaves HBM
// idle while it sums.  Here every thread fetches its vectors two to four rows ahead into slots of its own in shared
// memory (cp.async), so a row's sums run while the next rows arrive.  The arithmetic is done on pairs of f32
// (fma.rn.f32x2): at 8192 bf16 columns the plain form needs as many issue cycles as HBM needs time.
#pragma once

#include "kernels/block_norm_grad.cuh"
#include "kernels/pairs.cuh"

namespace afir {
namespace kernels {

// Rows of one team in order: its runs, each from begin to end.
struct RowCursor {
  int run, row, end, group;
  __device__ __forceinline__ void enter(const GradPlan &plan, int rows, int r) {
    run = r;
    if (run >= plan.groups * plan.chunks) {
      row = end = 0;
      return;
    }
    group = run / plan.chunks;
    const int chunk = run - group * plan.chunks;
    row = group * plan.groupRows + chunk * plan.chunkRows;
    end = min(min(rows - group * plan.groupRows, plan.groupRows), (chunk + 1) * plan.chunkRows) + group * plan.groupRows;
  }
  __device__ __forceinline__ bool live(const GradPlan &plan) const { return run < plan.groups * plan.chunks; }
  // On to a run that has rows (of a short last group the last runs have none).
  __device__ __forceinline__ void settle(const GradPlan &plan, int rows) {
    while (row >= end && live(plan)) enter(plan, rows, run + plan.teams);
  }
  __device__ __forceinline__ void advance(const GradPlan &plan, int rows) {
    ++row;
    settle(plan, rows);
  }
};

template <int ELEM, int KIND, int PASS, int NV>
__global__ void __launch_bounds__(512) blockNormGradVectorKernel(const __grid_constant__ BlockNormGradLaunch p, const __grid_constant__ GradPlan plan,
                                                                 int teamLanes, int stages) {
  gridDependencyPrologue();
  constexpr bool kLayer = KIND == kLayerNorm;
  constexpr int kValues = kLayer ? 2 : 1;
  constexpr bool kPostPart = PASS != kPre, kPrePart = PASS != kPost;
  constexpr int VEC = ElemOf<ELEM>::kVec, P = kPairs<ELEM>;
  extern __shared__ uint4 slots[];  // [stages][tensors][NV][threads]
  __shared__ float scratch[kTeamScratchFloats];
  Team team = makeTeam(teamLanes, scratch);
  const int cols = static_cast<int>(p.cols);
  const float share = 1.0f / static_cast<float>(cols);
  const int teamIndex = static_cast<int>(blockIdx.x) * team.count + team.index, rows = static_cast<int>(p.rows);
  if (teamIndex >= plan.teams) return;

  // which tensor has which slot
  const bool packed = p.checkpoint.codes != nullptr;
  const bool token = kPostPart && p.gateForm == kGateToken;
  int tensors = 0;
  const int slotDh = tensors;
  if (kPrePart) ++tensors;
  const int slotSource = tensors;
  if (kPrePart) ++tensors;
  const int slotDout = tensors;
  if (p.dout.base) ++tensors;
  const int slotY = tensors;
  if (kPostPart) ++tensors;
  const int slotGate = tensors;
  if (token) ++tensors;
  const int threads = static_cast<int>(blockDim.x);
  auto slot = [&](int stage, int tensor, int i) -> uint4 * { return slots + ((stage * tensors + tensor) * NV + i) * threads + threadIdx.x; };
  auto colOf = [&](int i) { return (i * team.lanes + team.lane) * VEC; };

  auto fetch = [&](const RowCursor &c, int stage) {
    if (c.live(plan)) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = colOf(i);
        if (col >= cols) continue;
        constexpr int eb = 16 / VEC;
        auto vectors = [&](int tensor, const RowsIn &r) { copyAhead16(slot(stage, tensor, i), static_cast<const char *>(r.base) + (static_cast<int64_t>(c.row) * r.ld + col) * eb); };
        auto codes = [&](int tensor) {
          const uint8_t *from = p.checkpoint.codes + static_cast<int64_t>(c.row) * p.checkpoint.codesLd + col;
          if constexpr (VEC == 8) copyAhead8(slot(stage, tensor, i), from);
          else copyAhead4(slot(stage, tensor, i), from);
        };
        if constexpr (kPrePart) {
          vectors(slotDh, p.dh);
          if (PASS == kPre && packed) codes(slotSource);
          else vectors(slotSource, p.source);
        }
        if (p.dout.base) vectors(slotDout, p.dout);
        if constexpr (kPostPart) {
          if (packed) codes(slotY);
          else vectors(slotY, p.y);
        }
        if (token) vectors(slotGate, p.gate);
      }
    }
    copiesCommit();  // an empty group where there is no row: the count stays the number of rows ahead
  };
  // what a row has besides its vectors, fetched one row ahead
  struct RowScalars { float rstdB, meanB, rstdA, meanA; int exps[NV]; };
  auto fetchScalars = [&](const RowCursor &c, RowScalars &s) {
    if (!c.live(plan)) return;
    if constexpr (kPrePart) {
      s.rstdB = __ldg(p.statsB.rstd + c.row);
      if constexpr (kLayer) s.meanB = __ldg(p.statsB.mean + c.row);
    }
    if constexpr (kPostPart) {
      s.rstdA = __ldg(p.statsA.rstd + c.row);
      if constexpr (kLayer) s.meanA = __ldg(p.statsA.mean + c.row);
    }
    if (packed) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (colOf(i) < cols) s.exps[i] = __ldg(p.checkpoint.exps + static_cast<int64_t>(c.row) * p.checkpoint.expsLd + colOf(i) / kCheckpointBlock);
    }
  };

  RowCursor now, ahead;
  now.enter(plan, rows, teamIndex);
  now.settle(plan, rows);
  ahead = now;
  RowScalars next = {};
  fetchScalars(now, next);
  for (int s = 0; s < stages; ++s) {
    fetch(ahead, s);
    ahead.advance(plan, rows);
  }

  const F2 zero = splat(0.0f);
  F2 sumB[kPrePart ? kValues : 1][NV][P], sumA[kPostPart ? kValues : 1][NV][P];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < P; ++e) {
#pragma unroll
      for (int k = 0; k < (kPrePart ? kValues : 1); ++k) sumB[k][i][e] = zero;
#pragma unroll
      for (int k = 0; k < (kPostPart ? kValues : 1); ++k) sumA[k][i][e] = zero;
    }
  auto storeSumPairs = [&](float *to, const F2 (&v)[P]) {
#pragma unroll
    for (int e = 0; e < P / 2; ++e) {
      const float2 a = valuesOf(v[2 * e]), b = valuesOf(v[2 * e + 1]);
      reinterpret_cast<float4 *>(to)[e] = make_float4(a.x, a.y, b.x, b.y);
    }
  };

  if constexpr (kPostPart) {  // runs without rows: sums of nothing
    RowCursor c;
    for (c.enter(plan, rows, teamIndex); c.live(plan); c.enter(plan, rows, c.run + plan.teams)) {
      if (c.row < c.end) continue;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < kValues; ++k)
          if (colOf(i) < cols) storeSumPairs(plan.sumsA + (static_cast<int64_t>(c.run) * kValues + k) * plan.sumsLd + colOf(i), sumA[k][i]);
    }
  }

  int stage = 0;
  while (now.live(plan)) {
    const RowScalars at = next;
    const int row = now.row, run = now.run, group = now.group;
    now.advance(plan, rows);
    fetchScalars(now, next);
    copiesWait(stages - 1);

    F2 dz[NV][P], n[NV][P];
    if constexpr (kPrePart) {
      const F2 rstd = splat(at.rstdB), shift = splat(kLayer ? -at.meanB : 0.0f);
      F2 s[kValues];
#pragma unroll
      for (int k = 0; k < kValues; ++k) s[k] = zero;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (colOf(i) >= cols) continue;
        F2 w[P];
        if (PASS == kPre && packed) codePairs<ELEM>(*reinterpret_cast<const uint2 *>(slot(stage, slotSource, i)), at.exps[i], n[i]);
        else widenPairs<ELEM>(*slot(stage, slotSource, i), n[i]);
        widenPairs<ELEM>(*slot(stage, slotDh, i), dz[i]);
        loadParamPairs<ELEM>(p.b.weight, p.paramType, colOf(i), w);
#pragma unroll
        for (int e = 0; e < P; ++e) {
          n[i][e] = kLayer ? (n[i][e] + shift) * rstd : n[i][e] * rstd;
          sumB[0][i][e] = fma2(dz[i][e], n[i][e], sumB[0][i][e]);
          if constexpr (kLayer) sumB[1][i][e] = sumB[1][i][e] + dz[i][e];
          dz[i][e] = dz[i][e] * w[e];
          s[0] = fma2(dz[i][e], n[i][e], s[0]);
          if constexpr (kLayer) s[1] = s[1] + dz[i][e];
        }
      }
      float total[kValues];
#pragma unroll
      for (int k = 0; k < kValues; ++k) total[k] = sumOf(s[k]);
      teamSum(team, total);
      const F2 along = splat(-total[0] * share * at.rstdB);
      const F2 constant = splat(kLayer ? -total[kValues - 1] * share * at.rstdB : 0.0f);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (colOf(i) >= cols) continue;
        F2 t[P];
        if (p.dout.base) widenPairs<ELEM>(*slot(stage, slotDout, i), t);
        else {
#pragma unroll
          for (int e = 0; e < P; ++e) t[e] = zero;
        }
#pragma unroll
        for (int e = 0; e < P; ++e) {
          if constexpr (kLayer) t[e] = t[e] + constant;
          dz[i][e] = fma2(dz[i][e], rstd, fma2(n[i][e], along, t[e]));
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (colOf(i) < cols) widenPairs<ELEM>(*slot(stage, slotDout, i), dz[i]);
    }

    if constexpr (!kPostPart) {
      fetch(ahead, stage);
      ahead.advance(plan, rows);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (colOf(i) < cols) storePairs<ELEM>(p.dx.base, static_cast<int64_t>(row) * p.dx.ld + colOf(i), dz[i]);
    } else {
      const F2 rstd = splat(at.rstdA), shift = splat(kLayer ? -at.meanA : 0.0f), alpha = splat(p.alpha);
      F2 s[kValues];
#pragma unroll
      for (int k = 0; k < kValues; ++k) s[k] = zero;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = colOf(i);
        if (col >= cols) continue;
        F2 t[P], w[P];
        if (packed) codePairs<ELEM>(*reinterpret_cast<const uint2 *>(slot(stage, slotY, i)), at.exps[i], n[i]);
        else widenPairs<ELEM>(*slot(stage, slotY, i), n[i]);
#pragma unroll
        for (int e = 0; e < P; ++e) {
          n[i][e] = kLayer ? (n[i][e] + shift) * rstd : n[i][e] * rstd;
          t[e] = dz[i][e] * alpha;
        }
        storePairs<ELEM>(p.dx.base, static_cast<int64_t>(row) * p.dx.ld + col, t);
        loadParamPairs<ELEM>(p.a.weight, p.paramType, col, w);
        F2 scale[P];
        if (p.scale) loadParamPairs<ELEM>(p.scale, p.paramType, col, scale);
        else {
#pragma unroll
          for (int e = 0; e < P; ++e) scale[e] = splat(1.0f);
        }
        if (p.gateForm == kGateNone) {
#pragma unroll
          for (int e = 0; e < P; ++e) {
            sumA[0][i][e] = fma2(dz[i][e], n[i][e], sumA[0][i][e]);
            if constexpr (kLayer) sumA[1][i][e] = sumA[1][i][e] + dz[i][e];
            dz[i][e] = dz[i][e] * (scale[e] * w[e]);
          }
        } else {
          F2 a[P];
          if (token) widenPairs<ELEM>(*slot(stage, slotGate, i), a);
          else loadPairs<ELEM>(p.gate.base, static_cast<int64_t>(group) * p.gate.ld + col, a);
          gatePairs(a, p.gateAct);
          if (token) {
            F2 u[P];
            if constexpr (kLayer) loadParamPairs<ELEM>(p.a.bias, p.paramType, col, u);
#pragma unroll
            for (int e = 0; e < P; ++e) {
              u[e] = kLayer ? fma2(n[i][e], w[e], u[e]) : n[i][e] * w[e];
              t[e] = dz[i][e] * scale[e] * u[e] * gateSlopePair(a[e], p.gateAct);
            }
            storePairs<ELEM>(p.dgate.base, static_cast<int64_t>(row) * p.dgate.ld + col, t);
          }
#pragma unroll
          for (int e = 0; e < P; ++e) {
            const F2 gated = dz[i][e] * a[e], forSums = token ? gated : dz[i][e];
            sumA[0][i][e] = fma2(forSums, n[i][e], sumA[0][i][e]);
            if constexpr (kLayer) sumA[1][i][e] = sumA[1][i][e] + forSums;
            dz[i][e] = gated * (scale[e] * w[e]);
          }
        }
#pragma unroll
        for (int e = 0; e < P; ++e) {
          s[0] = fma2(dz[i][e], n[i][e], s[0]);
          if constexpr (kLayer) s[1] = s[1] + dz[i][e];
        }
      }
      fetch(ahead, stage);  // this row's slots have been read
      ahead.advance(plan, rows);
      float total[kValues];
#pragma unroll
      for (int k = 0; k < kValues; ++k) total[k] = sumOf(s[k]);
      teamSum(team, total);
      const F2 along = splat(-total[0] * share * at.rstdA);
      const F2 constant = splat(kLayer ? -total[kValues - 1] * share * at.rstdA : 0.0f);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (colOf(i) >= cols) continue;
#pragma unroll
        for (int e = 0; e < P; ++e) {
          F2 t = kLayer ? fma2(n[i][e], along, constant) : n[i][e] * along;
          n[i][e] = fma2(dz[i][e], rstd, t);
        }
        storePairs<ELEM>(p.dy.base, static_cast<int64_t>(row) * p.dy.ld + colOf(i), n[i]);
      }
      if (now.run != run) {  // the run ends here: leave its sums and begin the next one's
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (colOf(i) < cols) {
#pragma unroll
            for (int k = 0; k < kValues; ++k) storeSumPairs(plan.sumsA + (static_cast<int64_t>(run) * kValues + k) * plan.sumsLd + colOf(i), sumA[k][i]);
          }
#pragma unroll
          for (int k = 0; k < kValues; ++k)
#pragma unroll
            for (int e = 0; e < P; ++e) sumA[k][i][e] = zero;
        }
      }
    }
    stage = stage + 1 == stages ? 0 : stage + 1;
  }
  if constexpr (kPrePart) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (colOf(i) >= cols) continue;
#pragma unroll
      for (int k = 0; k < kValues; ++k) storeSumPairs(plan.sumsB + (static_cast<int64_t>(teamIndex) * kValues + k) * plan.sumsLd + colOf(i), sumB[k][i]);
    }
  }
}

} // namespace kernels
} // namespace afir
