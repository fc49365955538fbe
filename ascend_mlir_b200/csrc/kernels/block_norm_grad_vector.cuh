// The gradient row kernel for rows in 16-byte vectors (formulas and the split of the rows: block_norm_grad.cuh).
//
// A row of the longest form is five tensors in and three out, so a team that loads when it needs the data leaves HBM
// idle while it sums.  Here every thread fetches its vectors two to four rows ahead into slots of its own in shared
// memory (cp.async), so a row's sums run while the next rows arrive.  The parameter vectors are kept there too: beside the
// rows they would not stay in what is left of the L1 (15 % hits), and every pass would wait for L2.  The arithmetic is done on
// pairs of f32 (fma.rn.f32x2): at 8192 bf16 columns the plain form needs as many issue cycles as HBM needs time.
//
// Measured without the joining kernel: 8192 x 8192 bf16 rms, a gate per element, both norms 174 us (1.07 GB, 6.2 TB/s: 94 % of a
// plain copy's rate); 8192 x 4096 bf16 rms from a checkpoint 42 us (235 MB, 5.6 TB/s); 4096 x 1024 f16 layer, a gate row per
// sequence 21.5 us (50 MB): seven rows per team, start-up and the column sums, which are a third of the bytes;
// 1023 x 1000 f32 layer 8.5 us.
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

// TOKEN: a gate value per element (kGateToken); FULL: every thread's vectors lie inside the row.
template <int ELEM, int KIND, int PASS, bool TOKEN, bool FULL, int NV>
__global__ void __launch_bounds__(kGradAheadThreads) blockNormGradVectorKernel(const __grid_constant__ BlockNormGradLaunch p, const __grid_constant__ GradPlan plan,
                                                                 int teamLanes, int stages) {
  gridDependencyPrologue();
  constexpr bool kLayer = KIND == kLayerNorm;
  constexpr int kValues = kLayer ? 2 : 1;
  constexpr bool kPostPart = PASS != kPre, kPrePart = PASS != kPost, kToken = TOKEN;
  constexpr int VEC = ElemOf<ELEM>::kVec, P = kPairs<ELEM>, EB = 16 / VEC;
  extern __shared__ uint4 slots[];  // [stages][tensors][NV][kGradAheadThreads], then parameters
  __shared__ TeamScratch scratch;
  Team team = makeTeam(teamLanes, scratch);
  const int cols = static_cast<int>(p.cols);
  const float share = 1.0f / static_cast<float>(cols);
  const int teamIndex = static_cast<int>(blockIdx.x) * team.count + team.index, rows = static_cast<int>(p.rows);
  if (teamIndex >= plan.teams) return;

  // A thread's columns: VEC from col0, and again every `apart` columns.
  const int col0 = team.lane * VEC, apart = team.lanes * VEC;
  bool has[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) has[i] = FULL || col0 + i * apart < cols;

  // Slots by byte: tensors present get one each, in this order.
  const bool grouped = !kToken && p.gateForm == kGateGroup;
  const bool packed = p.checkpoint.codes != nullptr, hasDout = p.dout.base != nullptr;
  constexpr unsigned int perVector = kGradAheadThreads * 16, perTensor = NV * perVector;
  unsigned int used = 0;
  const unsigned int atDh = used;
  if (kPrePart) used += perTensor;
  const unsigned int atSource = used;
  if (kPrePart) used += perTensor;
  const unsigned int atDout = used;
  if (hasDout) used += perTensor;
  const unsigned int atY = used;
  if (kPostPart) used += perTensor;
  const unsigned int atGate = used;
  if (kToken) used += perTensor;
  const unsigned int slot0 = threadIdx.x * 16, slotEnd = slot0 + stages * used;
  const unsigned int slotsAt = static_cast<unsigned int>(__cvta_generic_to_shared(slots));
  auto readSlot = [&](unsigned int at) { return *reinterpret_cast<const uint4 *>(reinterpret_cast<const char *>(slots) + at); };

  // Parameters as f32 behind the slots, each thread's own: normB's weight, normA's weight times the residual scale (and the
  // gate of the group that the team is in), and, where a token's gate needs it, normA's bias times the scale.
  constexpr unsigned int kParamFloats = NV * VEC * kGradAheadThreads;
  float *weightB = reinterpret_cast<float *>(reinterpret_cast<char *>(slots) + stages * used) + threadIdx.x * 4;
  float *weightA = weightB + (kPrePart ? kParamFloats : 0), *biasA = weightA + (kPostPart ? kParamFloats : 0);
  auto writeParams = [&](float *to, const void *v, const void *times, int gateRow = -1) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!has[i]) continue;
      F2 x[P], y[P];
      loadParamPairs<ELEM>(v, p.paramType, col0 + i * apart, x);
      if (times) {
        loadParamPairs<ELEM>(times, p.paramType, col0 + i * apart, y);
#pragma unroll
        for (int e = 0; e < P; ++e) x[e] = x[e] * y[e];
      }
      if (gateRow >= 0) {
        loadPairs<ELEM>(p.gate.base, static_cast<int64_t>(gateRow) * p.gate.ld + col0 + i * apart, y);
        gatePairs<ELEM>(y, p.gateAct);
#pragma unroll
        for (int e = 0; e < P; ++e) x[e] = x[e] * y[e];
      }
#pragma unroll
      for (int e = 0; e < P / 2; ++e) {
        const F2 quad[2] = {x[2 * e], x[2 * e + 1]};
        *reinterpret_cast<uint4 *>(to + (i * (P / 2) + e) * (kGradAheadThreads * 4)) = narrowPairs<kF32>(quad);
      }
    }
  };
  auto readParams = [&](const float *from, int i, F2 (&v)[P]) {
#pragma unroll
    for (int e = 0; e < P / 2; ++e) {
      F2 quad[2];
      widenPairs<kF32>(*reinterpret_cast<const uint4 *>(from + (i * (P / 2) + e) * (kGradAheadThreads * 4)), quad);
      v[2 * e] = quad[0];
      v[2 * e + 1] = quad[1];
    }
  };

  auto rowOf = [&](const RowsIn &r, int row) { return static_cast<const char *>(r.base) + (static_cast<int64_t>(row) * static_cast<int>(r.ld) + col0) * EB; };  // ld < 2^24
  auto rowTo = [&](const RowsOut &r, int row) { return static_cast<char *>(r.base) + (static_cast<int64_t>(row) * static_cast<int>(r.ld) + col0) * EB; };
  auto store = [&](char *to, int i, const F2 (&v)[P]) { *reinterpret_cast<uint4 *>(to + i * apart * EB) = narrowPairs<ELEM>(v); };

  auto fetch = [&](const RowCursor &c, unsigned int slot) {
    if (c.live(plan)) {
      auto vectors = [&](unsigned int at, const RowsIn &r) {
        const char *from = rowOf(r, c.row);
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (has[i]) copyAhead16(slotsAt + slot + at + i * perVector, from + i * apart * EB);
      };
      auto codes = [&](unsigned int at) {
        const uint8_t *from = p.checkpoint.codes + static_cast<int64_t>(c.row) * static_cast<int>(p.checkpoint.codesLd) + col0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (!has[i]) continue;
          if constexpr (VEC == 8) copyAhead8(slotsAt + slot + at + i * perVector, from + i * apart);
          else copyAhead4(slotsAt + slot + at + i * perVector, from + i * apart);
        }
      };
      if constexpr (kPrePart) {
        vectors(atDh, p.dh);
        if (PASS == kPre && packed) codes(atSource);
        else vectors(atSource, p.source);
      }
      if (hasDout) vectors(atDout, p.dout);
      if constexpr (kPostPart) {
        if (packed) codes(atY);
        else vectors(atY, p.y);
      }
      if constexpr (kToken) vectors(atGate, p.gate);
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
        if (has[i]) s.exps[i] = __ldg(p.checkpoint.exps + static_cast<int64_t>(c.row) * static_cast<int>(p.checkpoint.expsLd) + (col0 + i * apart) / kCheckpointBlock);
    }
  };

  RowCursor now, ahead;
  now.enter(plan, rows, teamIndex);
  now.settle(plan, rows);
  ahead = now;
  RowScalars next = {};
  fetchScalars(now, next);
  for (unsigned int s = slot0; s < slotEnd; s += used) {
    fetch(ahead, s);
    ahead.advance(plan, rows);
  }

  if constexpr (kPrePart) writeParams(weightB, p.b.weight, nullptr);
  if constexpr (kPostPart) writeParams(weightA, p.a.weight, p.scale, grouped && now.live(plan) ? now.group : -1);
  if constexpr (kToken && kLayer) writeParams(biasA, p.a.bias, p.scale);

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
  auto storeRunSums = [&](int run) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < kValues; ++k)
        if (has[i]) storeSumPairs(plan.sumsA + (static_cast<int64_t>(run) * kValues + k) * plan.sumsLd + col0 + i * apart, sumA[k][i]);
  };

  if (kPostPart && grouped) {  // runs without rows, of a short last group: sums of nothing
    RowCursor c;
    for (c.enter(plan, rows, teamIndex); c.live(plan); c.enter(plan, rows, c.run + plan.teams))
      if (c.row >= c.end) storeRunSums(c.run);
  }

  const GateSlope slope = gateSlopeOf(p.gateAct);
  unsigned int slot = slot0;
  while (now.live(plan)) {
    const RowScalars at = next;
    const int row = now.row, run = now.run;
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
        if (!has[i]) continue;
        F2 w[P];
        const uint4 raw = readSlot(slot + atSource + i * perVector);
        if (PASS == kPre && packed) codePairs<ELEM>(make_uint2(raw.x, raw.y), at.exps[i], n[i]);
        else widenPairs<ELEM>(raw, n[i]);
        widenPairs<ELEM>(readSlot(slot + atDh + i * perVector), dz[i]);
        readParams(weightB, i, w);
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
        if (!has[i]) continue;
        if (hasDout) {
          F2 t[P];
          widenPairs<ELEM>(readSlot(slot + atDout + i * perVector), t);
#pragma unroll
          for (int e = 0; e < P; ++e) {
            if constexpr (kLayer) t[e] = t[e] + constant;
            dz[i][e] = fma2(dz[i][e], rstd, fma2(n[i][e], along, t[e]));
          }
        } else {
#pragma unroll
          for (int e = 0; e < P; ++e) dz[i][e] = fma2(dz[i][e], rstd, kLayer ? fma2(n[i][e], along, constant) : n[i][e] * along);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (has[i]) widenPairs<ELEM>(readSlot(slot + atDout + i * perVector), dz[i]);
    }

    if constexpr (!kPostPart) {
      fetch(ahead, slot);
      ahead.advance(plan, rows);
      char *to = rowTo(p.dx, row);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (has[i]) store(to, i, dz[i]);
    } else {
      const F2 rstd = splat(at.rstdA), shift = splat(kLayer ? -at.meanA : 0.0f), alpha = splat(p.alpha);
      F2 s[kValues];
#pragma unroll
      for (int k = 0; k < kValues; ++k) s[k] = zero;
      char *toDx = rowTo(p.dx, row), *toDgate = kToken ? rowTo(p.dgate, row) : nullptr;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (!has[i]) continue;
        F2 t[P], w[P];  // w: normA's weight times the residual scale
        const uint4 raw = readSlot(slot + atY + i * perVector);
        if (packed) codePairs<ELEM>(make_uint2(raw.x, raw.y), at.exps[i], n[i]);
        else widenPairs<ELEM>(raw, n[i]);
#pragma unroll
        for (int e = 0; e < P; ++e) {
          n[i][e] = kLayer ? (n[i][e] + shift) * rstd : n[i][e] * rstd;
          t[e] = dz[i][e] * alpha;
        }
        store(toDx, i, t);
        readParams(weightA, i, w);
        if constexpr (kToken) {
          F2 a[P], bias[P];
          widenPairs<ELEM>(readSlot(slot + atGate + i * perVector), a);
          gatePairs<ELEM>(a, p.gateAct);
          if constexpr (kLayer) readParams(biasA, i, bias);
#pragma unroll
          for (int e = 0; e < P; ++e) {
            const F2 gated = dz[i][e] * a[e];
            sumA[0][i][e] = fma2(gated, n[i][e], sumA[0][i][e]);
            if constexpr (kLayer) sumA[1][i][e] = sumA[1][i][e] + gated;
            t[e] = dz[i][e] * (kLayer ? fma2(n[i][e], w[e], bias[e]) : n[i][e] * w[e]) * slopeAt(slope, a[e]);
            dz[i][e] = gated * w[e];
          }
          store(toDgate, i, t);
        } else {
#pragma unroll
          for (int e = 0; e < P; ++e) {
            sumA[0][i][e] = fma2(dz[i][e], n[i][e], sumA[0][i][e]);
            if constexpr (kLayer) sumA[1][i][e] = sumA[1][i][e] + dz[i][e];
            dz[i][e] = dz[i][e] * w[e];
          }
        }
#pragma unroll
        for (int e = 0; e < P; ++e) {
          s[0] = fma2(dz[i][e], n[i][e], s[0]);
          if constexpr (kLayer) s[1] = s[1] + dz[i][e];
        }
      }
      fetch(ahead, slot);  // this row's slots have been read
      ahead.advance(plan, rows);
      float total[kValues];
#pragma unroll
      for (int k = 0; k < kValues; ++k) total[k] = sumOf(s[k]);
      teamSum(team, total);
      const F2 along = splat(-total[0] * share * at.rstdA);
      const F2 constant = splat(kLayer ? -total[kValues - 1] * share * at.rstdA : 0.0f);
      char *toDy = rowTo(p.dy, row);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (!has[i]) continue;
#pragma unroll
        for (int e = 0; e < P; ++e) n[i][e] = fma2(dz[i][e], rstd, kLayer ? fma2(n[i][e], along, constant) : n[i][e] * along);
        store(toDy, i, n[i]);
      }
      if (now.run != run) {  // the run ends here: leave its sums and begin the next one's
        storeRunSums(run);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int k = 0; k < kValues; ++k)
#pragma unroll
            for (int e = 0; e < P; ++e) sumA[k][i][e] = zero;
        if (grouped && now.live(plan)) writeParams(weightA, p.a.weight, p.scale, now.group);
      }
    }
    slot = slot + used == slotEnd ? slot0 : slot + used;
  }
  if constexpr (kPrePart) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!has[i]) continue;
#pragma unroll
      for (int k = 0; k < kValues; ++k) storeSumPairs(plan.sumsB + (static_cast<int64_t>(teamIndex) * kValues + k) * plan.sumsLd + col0 + i * apart, sumB[k][i]);
    }
  }
}

} // namespace kernels
} // namespace afir
