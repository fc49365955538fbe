// Gradients of the row passes.  With n = (v - mean) * rstd a normed row and g the gradient of n*weight + bias,
//     dn = g*weight,   dv = rstd * (dn - n*avg(dn*n) [- avg(dn) for a layer norm]),
//     dweight = sum over rows of g*n,   dbias = sum over rows of g.
// Behind the gated sum, with dz the whole gradient of `out` (its later uses plus what normB sends back) and
// a = act(gate):
//     dx = alpha*dz,   du = dz*scale*a  (gradient of normA's output),   dgate = dz*scale*u*act'(gate),
//     u = n*weight + bias.
// The column sums of normA need only two of them, P = sum(a*dz*n) and Q = sum(a*dz): dweight = scale*P,
// dbias = scale*Q, dscale = weight*P + bias*Q (Q only for a layer norm).  Where one gate row serves a group of rows the
// sums are kept per group without `a` (it is the group's constant), and dgate = act'*scale*(weight*P + bias*Q) comes
// from them too, so a broadcast gate costs no second pass over the rows.
//
// One team per row, walking a run of neighbouring rows with the column sums of its columns in registers (f32), so all
// row tensors cross HBM once.  Each team leaves its sums in the workspace; a second kernel adds them in a fixed order
// (no atomics: the same inputs give the same bits).
#pragma once

#include "kernels/loose.cuh"

namespace afir {
namespace kernels {

// How the rows are split over teams, and where their sums go.  Depends on sizes only, so that the workspace can be
// sized before any pointer is known.
struct GradPlan {
  int groups;             // gate groups whose sums are kept apart (1 unless kGateGroup)
  int groupRows;          // rows of a group (all rows unless kGateGroup)
  int chunks;             // runs of rows per group
  int chunkRows;          // rows of a run
  int teams;              // teams launched; each takes runs index, index + teams, ...
  int sumsLd;             // floats of one row of sums (cols, rounded up to 16 bytes)
  float *sumsA, *sumsB;   // [groups*chunks][values][sumsLd], [teams][values][sumsLd]
};

// Any width and alignment (loose.cuh); aligned rows too that are too wide for block_norm_grad_vector.cuh.  Elements beyond
// the row are zeros, as are the parameters read for them, so they add nothing to a row's sums; they are not stored.  A row's
// loads are waited for one after the other and the arithmetic is not paired: 8000 x 4001 from a bf16 checkpoint 183 us (1.3
// TB/s), gated f16 rms 435 us; aligned 8192 x 8192 rows take 677 us here, 185 with rows fetched ahead.
template <int ELEM, int KIND, int PASS, int NV>
__global__ void __launch_bounds__(512) blockNormGradKernel(const __grid_constant__ BlockNormGradLaunch p, const __grid_constant__ GradPlan plan,
                                                           int teamLanes) {
  gridDependencyPrologue();
  constexpr bool kLayer = KIND == kLayerNorm;
  constexpr int VEC = ElemOf<ELEM>::kVec, EB = 16 / VEC;
  constexpr int kValues = kLayer ? 2 : 1;
  constexpr bool kPostPart = PASS != kPre, kPrePart = PASS != kPost;
  __shared__ TeamScratch scratch;
  Team team = makeTeam(teamLanes, scratch);
  const int cols = static_cast<int>(p.cols);
  const float share = 1.0f / static_cast<float>(cols);
  const int teamIndex = static_cast<int>(blockIdx.x) * team.count + team.index;
  if (teamIndex >= plan.teams) return;

  float sumB[kPrePart ? kValues : 1][NV][VEC];
#pragma unroll
  for (int k = 0; k < (kPrePart ? kValues : 1); ++k)
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) sumB[k][i][e] = 0.0f;

  for (int run = teamIndex; run < plan.groups * plan.chunks; run += plan.teams) {
    const int group = run / plan.chunks, chunk = run - group * plan.chunks;
    const int64_t groupBegin = static_cast<int64_t>(group) * plan.groupRows;
    const int64_t begin = groupBegin + static_cast<int64_t>(chunk) * plan.chunkRows;
    const int64_t end = min(min(p.rows, groupBegin + plan.groupRows), begin + plan.chunkRows);

    float sumA[kPostPart ? kValues : 1][NV][VEC];
#pragma unroll
    for (int k = 0; k < (kPostPart ? kValues : 1); ++k)
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) sumA[k][i][e] = 0.0f;

    for (int64_t row = begin; row < end; ++row) {
      float dz[NV][VEC];  // gradient of the stream
      // ---- through normB
      if constexpr (kPrePart) {
        const float mean = kLayer ? p.statsB.mean[row] : 0.0f, rstd = p.statsB.rstd[row];
        const bool fromCodes = PASS == kPre && p.checkpoint.codes != nullptr;
        float n[NV][VEC];
        float s[kValues];
#pragma unroll
        for (int k = 0; k < kValues; ++k) s[k] = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int col = (i * team.lanes + team.lane) * VEC;
          if (col >= cols) continue;
          float w[VEC];
          if (fromCodes) looseCheckpoint<VEC>(p.checkpoint, row, col, cols, innerRow(row, p.rows, p.checkpoint.codesLd), n[i]);
          else looseLoad<ELEM, VEC>(p.source.base, row * p.source.ld, col, cols, innerRow(row, p.rows, p.source.ld * EB), n[i]);
          looseLoad<ELEM, VEC>(p.dh.base, row * p.dh.ld, col, cols, innerRow(row, p.rows, p.dh.ld * EB), dz[i]);
          looseParam<ELEM, VEC>(p.b.weight, p.paramType, col, cols, w);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            n[i][e] = (n[i][e] - mean) * rstd;
            sumB[0][i][e] += dz[i][e] * n[i][e];
            if constexpr (kLayer) sumB[1][i][e] += dz[i][e];
            dz[i][e] *= w[e];
            s[0] += dz[i][e] * n[i][e];
            if constexpr (kLayer) s[1] += dz[i][e];
          }
        }
        teamSum(team, s);
        const float along = s[0] * share;
        float constant = 0.0f;
        if constexpr (kLayer) constant = s[1] * share;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int col = (i * team.lanes + team.lane) * VEC;
          if (col >= cols) continue;
#pragma unroll
          for (int e = 0; e < VEC; ++e) dz[i][e] = rstd * (dz[i][e] - n[i][e] * along - constant);
          if (p.dout.base) {
            float t[VEC];
            looseLoad<ELEM, VEC>(p.dout.base, row * p.dout.ld, col, cols, innerRow(row, p.rows, p.dout.ld * EB), t);
#pragma unroll
            for (int e = 0; e < VEC; ++e) dz[i][e] += t[e];
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int col = (i * team.lanes + team.lane) * VEC;
          if (col < cols) looseLoad<ELEM, VEC>(p.dout.base, row * p.dout.ld, col, cols, innerRow(row, p.rows, p.dout.ld * EB), dz[i]);
        }
      }
      if constexpr (!kPostPart) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int col = (i * team.lanes + team.lane) * VEC;
          if (col < cols) looseStore<ELEM, VEC>(p.dx.base, row * p.dx.ld, col, cols, dz[i]);
        }
      } else {
        // ---- through the gated sum and normA
        const float mean = kLayer ? p.statsA.mean[row] : 0.0f, rstd = p.statsA.rstd[row];
        const bool fromCodes = p.checkpoint.codes != nullptr;
        const bool token = p.gateForm == kGateToken;
        float n[NV][VEC];
        float s[kValues];
#pragma unroll
        for (int k = 0; k < kValues; ++k) s[k] = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int col = (i * team.lanes + team.lane) * VEC;
          if (col >= cols) continue;
          float t[VEC], a[VEC], scale[VEC], w[VEC];
          if (fromCodes) looseCheckpoint<VEC>(p.checkpoint, row, col, cols, innerRow(row, p.rows, p.checkpoint.codesLd), n[i]);
          else looseLoad<ELEM, VEC>(p.y.base, row * p.y.ld, col, cols, innerRow(row, p.rows, p.y.ld * EB), n[i]);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            n[i][e] = (n[i][e] - mean) * rstd;
            a[e] = 1.0f;
            scale[e] = 1.0f;
          }
          if (p.gateForm != kGateNone) {
            {
              const int64_t gateRow = token ? row : group;
              looseLoad<ELEM, VEC>(p.gate.base, gateRow * p.gate.ld, col, cols, innerRow(gateRow, token ? p.rows : plan.groups, p.gate.ld * EB), a);
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) a[e] = gateValue(a[e], p.gateAct);
          }
          if (p.scale) looseParam<ELEM, VEC>(p.scale, p.paramType, col, cols, scale);
          looseParam<ELEM, VEC>(p.a.weight, p.paramType, col, cols, w);
#pragma unroll
          for (int e = 0; e < VEC; ++e) t[e] = p.alpha * dz[i][e];
          looseStore<ELEM, VEC>(p.dx.base, row * p.dx.ld, col, cols, t);
          if (token) {
            float bias[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) bias[e] = 0.0f;
            if constexpr (kLayer) looseParam<ELEM, VEC>(p.a.bias, p.paramType, col, cols, bias);
#pragma unroll
            for (int e = 0; e < VEC; ++e) t[e] = dz[i][e] * scale[e] * fmaf(n[i][e], w[e], bias[e]) * gateSlope(a[e], p.gateAct);
            looseStore<ELEM, VEC>(p.dgate.base, row * p.dgate.ld, col, cols, t);
          }
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float forSums = token ? dz[i][e] * a[e] : dz[i][e];
            sumA[0][i][e] += forSums * n[i][e];
            if constexpr (kLayer) sumA[1][i][e] += forSums;
            dz[i][e] *= scale[e] * a[e] * w[e];
            s[0] += dz[i][e] * n[i][e];
            if constexpr (kLayer) s[1] += dz[i][e];
          }
        }
        teamSum(team, s);
        const float along = s[0] * share;
        float constant = 0.0f;
        if constexpr (kLayer) constant = s[1] * share;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int col = (i * team.lanes + team.lane) * VEC;
          if (col >= cols) continue;
          float t[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) t[e] = rstd * (dz[i][e] - n[i][e] * along - constant);
          looseStore<ELEM, VEC>(p.dy.base, row * p.dy.ld, col, cols, t);
        }
      }
    }
    if constexpr (kPostPart) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (i * team.lanes + team.lane) * VEC;
        if (col >= cols) continue;
#pragma unroll
        for (int k = 0; k < kValues; ++k) looseSums<VEC>(plan.sumsA + (static_cast<int64_t>(run) * kValues + k) * plan.sumsLd + col, col, cols, sumA[k][i]);
      }
    }
  }
  if constexpr (kPrePart) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * team.lanes + team.lane) * VEC;
      if (col >= cols) continue;
#pragma unroll
      for (int k = 0; k < kValues; ++k) looseSums<VEC>(plan.sumsB + (static_cast<int64_t>(teamIndex) * kValues + k) * plan.sumsLd + col, col, cols, sumB[k][i]);
    }
  }
}

} // namespace kernels
} // namespace afir
