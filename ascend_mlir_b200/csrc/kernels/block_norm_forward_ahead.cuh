// The forward row kernel for many rows in 16-byte vectors: teams that stay, rows fetched ahead.
//
// A row costs a thread about as many instructions besides its vectors (statistics across warps, addresses, set-up of the
// CTA) as two or three vectors do, and a kernel that starts a team for every row was bound by them.  Here a team walks
// every teams-th row with its set-up done once, its parameters in shared memory as f32 (scale folded into normA's), and the
// next rows arriving in slots of its threads (as in block_norm_grad_vector.cuh) while it sums.
//
// Measured: 8192 x 4096 bf16 rms with a checkpoint 32.7 us (168 MB, 5.1 TB/s: 78 % of a plain copy's rate; starts and last
// rows count at this size); 16384 x 4096 f16 layer, a gate row per sequence, both norms, 121 us (537 MB, 4.4 TB/s): bound by
// instruction issue (2.3 per cycle) and the shared memory that rows and parameters come from.
#pragma once

#include "kernels/block_norm_forward_vector.cuh"

namespace afir {
namespace kernels {

// FULL: every thread's vectors lie inside the row.
template <int ELEM, int KIND, int PASS, bool FULL, int NV>
__global__ void __launch_bounds__(PASS == kPre ? kForwardAheadThreads : kForwardAheadPostThreads, PASS == kPre ? 2 : 1) blockNormForwardAheadKernel(const __grid_constant__ BlockNormLaunch p, int teamLanes,
                                                                                          int stages) {
  gridDependencyPrologue();
  constexpr bool kLayer = KIND == kLayerNorm;
  constexpr int VEC = ElemOf<ELEM>::kVec, P = kPairs<ELEM>, EB = 16 / VEC;
  extern __shared__ uint4 slots[];  // [stages][tensors][NV][perVector / 16], then parameters
  __shared__ TeamScratch scratch;
  Team team = makeTeam(teamLanes, scratch);
  const int cols = static_cast<int>(p.cols), rows = static_cast<int>(p.rows);
  const float share = 1.0f / static_cast<float>(cols);
  const int step = static_cast<int>(gridDim.x) * team.count;
  int row = static_cast<int>(blockIdx.x) * team.count + team.index;
  if (row >= rows) return;

  const int col0 = team.lane * VEC, apart = team.lanes * VEC;
  bool has[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) has[i] = FULL || col0 + i * apart < cols;
  const bool gated = PASS != kPre && p.gateForm != kGateNone, grouped = PASS != kPre && p.gateForm == kGateGroup;
  const unsigned int groupRows = static_cast<unsigned int>(p.groupRows);  // at most the rows

  constexpr unsigned int perVector = (PASS == kPre ? kForwardAheadThreads : kForwardAheadPostThreads) * 16, perTensor = NV * perVector;
  constexpr unsigned int atX = PASS == kPre ? 0 : perTensor, atGate = 2 * perTensor;
  const unsigned int used = PASS == kPre ? perTensor : gated ? 3 * perTensor : 2 * perTensor;
  const unsigned int slot0 = threadIdx.x * 16, slotEnd = slot0 + stages * used;
  const unsigned int slotsAt = static_cast<unsigned int>(__cvta_generic_to_shared(slots));
  auto readSlot = [&](unsigned int at) { return *reinterpret_cast<const uint4 *>(reinterpret_cast<const char *>(slots) + at); };
  auto rowTo = [&](const RowsOut &r) { return static_cast<char *>(r.base) + (static_cast<int64_t>(row) * static_cast<int>(r.ld) + col0) * EB; };

  auto fetch = [&](int at, unsigned int slot) {
    if (at < rows) {
      auto vectors = [&](unsigned int where, const RowsIn &r, int which) {
        const char *from = static_cast<const char *>(r.base) + (static_cast<int64_t>(which) * static_cast<int>(r.ld) + col0) * EB;  // ld < 2^24
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (has[i]) copyAhead16(slotsAt + slot + where + i * perVector, from + i * apart * EB);
      };
      if constexpr (PASS != kPre) {
        vectors(0, p.y, at);
        if (gated) vectors(atGate, p.gate, grouped ? static_cast<int>(static_cast<unsigned int>(at) / groupRows) : at);
      }
      vectors(atX, p.x, at);
    }
    copiesCommit();  // an empty group where there is no row: the count stays the number of rows ahead
  };
  // (slots of vectors beyond the row are never filled and would be read as they are: they hold zeros)
  if constexpr (!FULL) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (!has[i])
        for (unsigned int at = slot0 + i * perVector; at < slotEnd; at += perTensor) *reinterpret_cast<uint4 *>(reinterpret_cast<char *>(slots) + at) = make_uint4(0u, 0u, 0u, 0u);
  }
  int ahead = row;
  for (unsigned int s = slot0; s < slotEnd; s += used, ahead += step) fetch(ahead, s);

  // Parameters of all teams of the CTA; a thread reads only what it has written itself (teams write the same values).
  // 16-byte pieces in the order of the threads, free of bank conflicts.
  const int paramLd = team.lanes * NV * VEC;
  float *weightA = reinterpret_cast<float *>(reinterpret_cast<char *>(slots) + stages * used);
  float *biasA = weightA + (PASS != kPre ? paramLd : 0), *weightB = biasA + (PASS != kPre && kLayer ? paramLd : 0);
  float *biasB = weightB + (PASS != kPost ? paramLd : 0);
  auto writeParams = [&](float *to, const void *v, const void *times) {
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
#pragma unroll
      for (int e = 0; e < P / 2; ++e) {
        const F2 quad[2] = {x[2 * e], x[2 * e + 1]};
        *reinterpret_cast<uint4 *>(to + ((i * (P / 2) + e) * team.lanes + team.lane) * 4) = narrowPairs<kF32>(quad);
      }
    }
  };
  auto readParams = [&](const float *from, int i, F2 (&v)[P]) {
#pragma unroll
    for (int e = 0; e < P / 2; ++e) {
      F2 quad[2];
      widenPairs<kF32>(*reinterpret_cast<const uint4 *>(from + ((i * (P / 2) + e) * team.lanes + team.lane) * 4), quad);
      v[2 * e] = quad[0];
      v[2 * e + 1] = quad[1];
    }
  };
  if constexpr (PASS != kPre) {
    writeParams(weightA, p.a.weight, p.scale);
    if constexpr (kLayer) writeParams(biasA, p.a.bias, p.scale);
  }
  if constexpr (PASS != kPost) {
    writeParams(weightB, p.b.weight, nullptr);
    if constexpr (kLayer) writeParams(biasB, p.b.bias, nullptr);
  }
  // v normed, times weight, plus bias
  auto normed = [&](F2 (&v)[P], int i, F2 shift, F2 rstd, const float *weight, const float *bias) {
    F2 w[P];
    readParams(weight, i, w);
    if constexpr (kLayer) {
      F2 b[P];
      readParams(bias, i, b);
#pragma unroll
      for (int e = 0; e < P; ++e) v[e] = fma2((v[e] + shift) * rstd, w[e], b[e]);
    } else {
#pragma unroll
      for (int e = 0; e < P; ++e) v[e] = v[e] * rstd * w[e];
    }
  };

  unsigned int slot = slot0;
  for (; row < rows; row += step, ahead += step) {
    copiesWait(stages - 1);
    F2 v[NV][P];
    uint4 first[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      first[i] = readSlot(slot + i * perVector);
      widenPairs<ELEM>(first[i], v[i]);
    }
    if (p.checkpoint.codes) {
#pragma unroll
      for (int i = 0; i < NV; ++i) packVector<ELEM>(first[i], has[i], col0 + i * apart, row, p.checkpoint);
    }
    if constexpr (PASS == kPre) fetch(ahead, slot);  // this row's slots have been read
    float mean, rstd;
    pairStatistics<ELEM, KIND, NV>(team, v, cols, share, FULL, PASS == kPre ? p.epsB : p.epsA, mean, rstd);
    storeStatistics(team, PASS == kPre ? p.statsB : p.statsA, row, mean, rstd);
    if constexpr (PASS != kPre) {
      const F2 shift = splat(-mean), r = splat(rstd), alpha = splat(p.alpha);
      char *to = rowTo(p.out);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (!has[i]) continue;
        normed(v[i], i, shift, r, weightA, biasA);
        F2 t[P];
        if (gated) {
          widenPairs<ELEM>(readSlot(slot + atGate + i * perVector), t);
          gatePairs<ELEM>(t, p.gateAct);
#pragma unroll
          for (int e = 0; e < P; ++e) v[i][e] = v[i][e] * t[e];
        }
        widenPairs<ELEM>(readSlot(slot + atX + i * perVector), t);
#pragma unroll
        for (int e = 0; e < P; ++e) v[i][e] = fma2(alpha, t[e], v[i][e]);
        const uint4 stored = narrowPairs<ELEM>(v[i]);
        *reinterpret_cast<uint4 *>(to + i * apart * EB) = stored;
        if constexpr (PASS == kPostPre) widenPairs<ELEM>(stored, v[i]);  // as it is stored
      }
      fetch(ahead, slot);
      if constexpr (PASS == kPostPre) {
        pairStatistics<ELEM, KIND, NV>(team, v, cols, share, FULL, p.epsB, mean, rstd);
        storeStatistics(team, p.statsB, row, mean, rstd);
      }
    }
    if constexpr (PASS != kPost) {
      const F2 shift = splat(-mean), r = splat(rstd);
      char *to = rowTo(p.h);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (!has[i]) continue;
        normed(v[i], i, shift, r, weightB, biasB);
        *reinterpret_cast<uint4 *>(to + i * apart * EB) = narrowPairs<ELEM>(v[i]);
      }
    }
    slot = slot + used == slotEnd ? slot0 : slot + used;
  }
}

} // namespace kernels
} // namespace afir
