// The forward row kernel for rows in 16-byte vectors (formulas: block_norm_forward.cuh).
//
// A thread issues the loads of everything it will need of a row (y, x and a token's gate) before the first sum, so that
// the sums wait for HBM once.  It is for few rows, where that one wait and the way from load to store are all the time there is:
// 1 x 4096 bf16 4.1 us, 16 gated rows of 8192 7.7 us.  A layer norm's statistics take one barrier: each warp centres its own columns, and the
// warps' sums of squares are joined with what their means differ by (Chan, Golub and LeVeque's update).
#pragma once

#include "kernels/block_norm_forward.cuh"
#include "kernels/pairs.cuh"

namespace afir {
namespace kernels {

// Of f32 rows rounded once; of 16-bit rows within two units in the last place of f32, in fewer instructions (16384 x 4096 f16
// layer, both norms: 114 us, 121 rounded once).
template <int ELEM> __device__ __forceinline__ float inverseRoot(float v) { return ELEM == kF32 ? __frsqrt_rn(v) : rsqrtf(v); }

// Mean and 1/sqrt(variance + eps) of the row in v; what lies beyond the row is zero in v and not counted.
template <int ELEM, int KIND, int NV>
__device__ __forceinline__ void pairStatistics(Team &team, const F2 (&v)[NV][kPairs<ELEM>], int cols, float share, bool full, float eps, float &mean, float &rstd) {
  constexpr int VEC = ElemOf<ELEM>::kVec, P = kPairs<ELEM>;
  if constexpr (KIND == kRmsNorm) {
    F2 q = splat(0.0f);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < P; ++e) q = fma2(v[i][e], v[i][e], q);
    float s[1] = {sumOf(q)};
    teamSum(team, s);
    mean = 0.0f;
    rstd = inverseRoot<ELEM>(s[0] * share + eps);
  } else {
    F2 sum = splat(0.0f);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < P; ++e) sum = sum + v[i][e];
    const float s = warpSum(sumOf(sum));
    float mine = static_cast<float>(NV * 32 * VEC);  // of the row, in this warp's lanes
    if (!full) {
      int n = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) n += max(0, min(32 * VEC, cols - (i * team.lanes + (team.lane & ~31)) * VEC));
      mine = static_cast<float>(n);
    }
    constexpr float kWhole = 1.0f / (NV * 32 * VEC);  // a power of two
    const float centre = full ? s * kWhole : __fdividef(s, fmaxf(mine, 1.0f));  // any centre near the mean will do
    const F2 shift = splat(-centre);
    F2 q = splat(0.0f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!full && (i * team.lanes + team.lane) * VEC >= cols) continue;
#pragma unroll
      for (int e = 0; e < P; ++e) {
        const F2 d = v[i][e] + shift;
        q = fma2(d, d, q);
      }
    }
    float squares = warpSum(sumOf(q));
    if (team.lanes == 32) {
      mean = s * share;
      squares = fmaf(mine * (centre - mean), centre - mean, squares);
    } else {
      float *buf = team.scratch + team.half * (kTeamValues * kTeamSlice);
      team.half ^= 1;
      if ((threadIdx.x & 31) == 0) {
        const int w = team.lane >> 5;
        buf[w] = s;
        buf[kTeamSlice + w] = squares;
        if (!full) buf[2 * kTeamSlice + w] = mine;
      }
      teamBarrier(team);
      // each warp joins the warps' sums in a shuffle tree over the next power of two of them
      const int warps = team.lanes >> 5, tree = warps <= 2 ? 2 : warps <= 4 ? 4 : warps <= 8 ? 8 : 16;
      const int w = threadIdx.x & (tree - 1);
      const float sw = buf[w], count = full ? (w < warps ? static_cast<float>(NV * 32 * VEC) : 0.0f) : buf[2 * kTeamSlice + w];
      auto treeSum = [&](float t) {
#pragma unroll
        for (int o = 8; o > 0; o >>= 1)
          if (o < tree) t += __shfl_xor_sync(0xffffffffu, t, o);
        return t;
      };
      mean = treeSum(sw) * share;
      const float off = (full ? sw * kWhole : __fdividef(sw, fmaxf(count, 1.0f))) - mean;  // the same quotient as the warp's centre
      squares = treeSum(fmaf(count * off, off, buf[kTeamSlice + w]));
    }
    rstd = inverseRoot<ELEM>(squares * share + eps);
  }
}

// v normed, times weight, plus bias.
template <int ELEM, int KIND>
__device__ __forceinline__ void normPairs(F2 (&v)[kPairs<ELEM>], F2 shift, F2 rstd, const NormVectors &p, int paramType, int col) {
  F2 w[kPairs<ELEM>];
  loadParamPairs<ELEM>(p.weight, paramType, col, w);
#pragma unroll
  for (int e = 0; e < kPairs<ELEM>; ++e) v[e] = (KIND == kLayerNorm ? (v[e] + shift) * rstd : v[e] * rstd) * w[e];
  if constexpr (KIND == kLayerNorm) {
    loadParamPairs<ELEM>(p.bias, paramType, col, w);
#pragma unroll
    for (int e = 0; e < kPairs<ELEM>; ++e) v[e] = v[e] + w[e];
  }
}

template <int ELEM, int KIND, int PASS, int NV>
__global__ void __launch_bounds__(512) blockNormForwardVectorKernel(const __grid_constant__ BlockNormLaunch p, int teamLanes) {
  gridDependencyPrologue();
  constexpr int VEC = ElemOf<ELEM>::kVec, P = kPairs<ELEM>;
  constexpr int kPostVectors = PASS == kPre ? 1 : NV;
  __shared__ TeamScratch scratch;
  Team team = makeTeam(teamLanes, scratch);
  const int cols = static_cast<int>(p.cols);
  const float share = 1.0f / static_cast<float>(cols);
  const bool full = team.lanes * NV * VEC == cols;
  const int64_t step = static_cast<int64_t>(gridDim.x) * team.count;
  auto colOf = [&](int i) { return (i * team.lanes + team.lane) * VEC; };
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * team.count + team.index; row < p.rows; row += step) {
    const RowsIn first = PASS == kPre ? p.x : p.y;
    auto raw = [&](const RowsIn &r, int64_t at, int i) {
      return *reinterpret_cast<const uint4 *>(static_cast<const char *>(r.base) + (at * r.ld + colOf(i)) * (16 / VEC));
    };
    uint4 raw0[NV], rawX[kPostVectors], rawGate[kPostVectors];
    const bool gated = PASS != kPre && p.gateForm != kGateNone;
    int64_t gateRow = row;  // rows and groups are counted in 32 bits
    if (PASS != kPre && p.gateForm == kGateGroup)
      gateRow = static_cast<unsigned int>(row) / static_cast<unsigned int>(p.groupRows);
#pragma unroll
    for (int i = 0; i < NV; ++i) raw0[i] = colOf(i) < cols ? raw(first, row, i) : make_uint4(0u, 0u, 0u, 0u);
    if constexpr (PASS != kPre) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (colOf(i) >= cols) continue;
        rawX[i] = raw(p.x, row, i);
        if (gated) rawGate[i] = raw(p.gate, gateRow, i);
      }
    }
    F2 v[NV][P];
#pragma unroll
    for (int i = 0; i < NV; ++i) widenPairs<ELEM>(raw0[i], v[i]);
    if (p.checkpoint.codes) {
#pragma unroll
      for (int i = 0; i < NV; ++i) packVector<ELEM>(raw0[i], colOf(i) < cols, colOf(i), row, p.checkpoint);
    }
    float mean, rstd;
    pairStatistics<ELEM, KIND, NV>(team, v, cols, share, full, PASS == kPre ? p.epsB : p.epsA, mean, rstd);
    storeStatistics(team, PASS == kPre ? p.statsB : p.statsA, row, mean, rstd);
    if constexpr (PASS != kPre) {
      const F2 shift = splat(-mean), r = splat(rstd), alpha = splat(p.alpha);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = colOf(i);
        if (col >= cols) continue;
        normPairs<ELEM, KIND>(v[i], shift, r, p.a, p.paramType, col);
        F2 t[P];
        if (gated) {
          widenPairs<ELEM>(rawGate[i], t);
          gatePairs<ELEM>(t, p.gateAct);
#pragma unroll
          for (int e = 0; e < P; ++e) v[i][e] = v[i][e] * t[e];
        }
        if (p.scale) {
          loadParamPairs<ELEM>(p.scale, p.paramType, col, t);
#pragma unroll
          for (int e = 0; e < P; ++e) v[i][e] = v[i][e] * t[e];
        }
        widenPairs<ELEM>(rawX[i], t);
#pragma unroll
        for (int e = 0; e < P; ++e) v[i][e] = fma2(alpha, t[e], v[i][e]);
        const uint4 stored = narrowPairs<ELEM>(v[i]);
        *reinterpret_cast<uint4 *>(static_cast<char *>(p.out.base) + (row * p.out.ld + col) * (16 / VEC)) = stored;
        if constexpr (PASS == kPostPre) widenPairs<ELEM>(stored, v[i]);  // as it is stored
      }
      if constexpr (PASS == kPostPre) {
        pairStatistics<ELEM, KIND, NV>(team, v, cols, share, full, p.epsB, mean, rstd);
        storeStatistics(team, p.statsB, row, mean, rstd);
      }
    }
    if constexpr (PASS != kPost) {
      const F2 shift = splat(-mean), r = splat(rstd);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = colOf(i);
        if (col >= cols) continue;
        normPairs<ELEM, KIND>(v[i], shift, r, p.b, p.paramType, col);
        storePairs<ELEM>(p.h.base, row * p.h.ld + col, v[i]);
      }
    }
  }
}

} // namespace kernels
} // namespace afir
