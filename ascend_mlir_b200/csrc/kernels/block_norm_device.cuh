// Device pieces shared by the row passes (block_norm_forward.cuh, block_norm_grad.cuh) and the checkpoint kernels:
// vectors of 16 bytes widened to f32, teams of threads that own one row, and the 8-bit format.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "kernels/block_norm.h"
#include "kernels/grid_dependency.cuh"

namespace afir {
namespace kernels {

// ---- elements ---------------------------------------------------------------------------------------------------
template <int ELEM> struct ElemOf;
template <> struct ElemOf<kF32> {
  using Type = float;
  static constexpr int kVec = 4;  // elements in 16 bytes
  __device__ __forceinline__ static float widen(float v) { return v; }
  __device__ __forceinline__ static float narrow(float v) { return v; }
};
template <> struct ElemOf<kF16> {
  using Type = __half;
  static constexpr int kVec = 8;
  __device__ __forceinline__ static float widen(__half v) { return __half2float(v); }
  __device__ __forceinline__ static __half narrow(float v) { return __float2half_rn(v); }
};
template <> struct ElemOf<kBF16> {
  using Type = __nv_bfloat16;
  static constexpr int kVec = 8;
  __device__ __forceinline__ static float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
  __device__ __forceinline__ static __nv_bfloat16 narrow(float v) { return __float2bfloat16_rn(v); }
};

template <int ELEM, int VEC> __device__ __forceinline__ void unpack(const uint4 &raw, float (&v)[VEC]) {
  static_assert(VEC == ElemOf<ELEM>::kVec, "16 bytes");
  const unsigned int w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (ELEM == kF32) v[i] = __uint_as_float(w[i]);
    else if constexpr (ELEM == kF16) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    } else {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}
template <int ELEM, int VEC> __device__ __forceinline__ uint4 pack(const float (&v)[VEC]) {
  static_assert(VEC == ElemOf<ELEM>::kVec, "16 bytes");
  unsigned int w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (ELEM == kF32) w[i] = __float_as_uint(v[i]);
    else if constexpr (ELEM == kF16) {
      const __half2 p = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const unsigned int *>(&p);
    } else {
      const __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const unsigned int *>(&p);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// VEC elements at `p` (16-byte aligned when VEC > 1), widened.
template <int ELEM, int VEC> __device__ __forceinline__ void loadElems(const void *p, int64_t at, float (&v)[VEC]) {
  using T = typename ElemOf<ELEM>::Type;
  const T *q = static_cast<const T *>(p) + at;
  if constexpr (VEC == 1) v[0] = ElemOf<ELEM>::widen(*q);
  else unpack<ELEM, VEC>(*reinterpret_cast<const uint4 *>(q), v);
}
// A parameter vector, or one parameter: of the rows' type or f32 (uniform over the launch); it stays in L1 from row to row.
template <int ELEM, int VEC> __device__ __forceinline__ void loadParam(const void *p, int type, int at, float (&v)[VEC]) {
  if (ELEM == kF32 || type != kF32) {
    loadElems<ELEM, VEC>(p, at, v);
  } else if constexpr (VEC == 1) {
    v[0] = static_cast<const float *>(p)[at];
  } else {
    const float4 *q = reinterpret_cast<const float4 *>(static_cast<const float *>(p) + at);
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      const float4 f = q[i];
      v[4 * i] = f.x;
      v[4 * i + 1] = f.y;
      v[4 * i + 2] = f.z;
      v[4 * i + 3] = f.w;
    }
  }
}

// ---- teams ------------------------------------------------------------------------------------------------------
// `lanes` threads (a multiple of 32, at most 512) that hold one row; a CTA of up to 1024 threads has one or more of them
// (at most 15 of more than a warp: each has a named barrier).  Sums over a team: a shuffle tree in each warp, then the
// warps' sums through shared memory, which every thread of up to 8 warps adds up itself in the same order (a second shuffle
// tree would be five more dependent latencies); of more warps, each warp adds them in a shuffle tree.  The two halves of the
// buffer alternate, so one barrier per sum is enough: whoever writes a half again has passed the barrier of the sum between,
// which every reader of that half reached after reading.
struct Team {
  int lanes, lane, index, count;  // threads in it; this thread's place; which of the CTA's; how many the CTA has
  float *scratch;                 // this team's slice of the CTA's buffer: [halves][kTeamValues][slice], zero beyond its warps
  int half;
};
constexpr int kTeamValues = 3;
constexpr int kTeamSlice = 64;  // floats per value: the CTA's warps, each team's rounded up to 4, 8 or 16
constexpr int kTeamScratchFloats = 2 * kTeamValues * kTeamSlice;
struct alignas(16) TeamScratch { float values[kTeamScratchFloats]; };  // the CTA's buffer: read 16 bytes at a time

__device__ __forceinline__ void teamBarrier(const Team &t) { asm volatile("bar.sync %0, %1;" ::"r"(t.index + 1), "r"(t.lanes) : "memory"); }

__device__ __forceinline__ Team makeTeam(int lanes, TeamScratch &scratch) {
  Team t;
  t.lanes = lanes;
  t.index = static_cast<int>(threadIdx.x) / lanes;
  t.lane = static_cast<int>(threadIdx.x) - t.index * lanes;
  t.count = static_cast<int>(blockDim.x) / lanes;
  const int warps = lanes >> 5, slice = warps <= 4 ? 4 : warps <= 8 ? 8 : 16;
  t.scratch = scratch.values + t.index * slice;
  t.half = 0;
  if (lanes > 32) {
    if (t.lane < slice) {
#pragma unroll
      for (int v = 0; v < 2 * kTeamValues; ++v) t.scratch[v * kTeamSlice + t.lane] = 0.0f;
    }
    teamBarrier(t);
  }
  return t;
}
__device__ __forceinline__ float warpSum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int N> __device__ __forceinline__ void teamSum(Team &t, float (&v)[N]) {
  static_assert(N <= kTeamValues, "the buffer holds that many values per warp");
#pragma unroll
  for (int n = 0; n < N; ++n) v[n] = warpSum(v[n]);
  if (t.lanes == 32) return;
  float *buf = t.scratch + t.half * (kTeamValues * kTeamSlice);
  t.half ^= 1;
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int n = 0; n < N; ++n) buf[n * kTeamSlice + (t.lane >> 5)] = v[n];
  }
  teamBarrier(t);
  if (t.lanes <= 256) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const float4 a = *reinterpret_cast<const float4 *>(buf + n * kTeamSlice);
      v[n] = (a.x + a.y) + (a.z + a.w);
      if (t.lanes > 128) {
        const float4 b = *reinterpret_cast<const float4 *>(buf + n * kTeamSlice + 4);
        v[n] += (b.x + b.y) + (b.z + b.w);
      }
    }
  } else {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      v[n] = lane < (t.lanes >> 5) ? buf[n * kTeamSlice + lane] : 0.0f;
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
      v[n] = __shfl_sync(0xffffffffu, v[n], 0);
    }
  }
}

// ---- the 8-bit format -------------------------------------------------------------------------------------------
// Exponent of the power of two for a block whose largest finite magnitude is `top`: the smallest with
// top <= 448 * 2^(e - 127), kept where the restored values fit the type: down to the power whose smallest code
// (2^-9 of it) is the type's last subnormal bit or coarser, up to the one that needs codes beyond 240 cut
// (256 * that power would be past the type's largest value).
template <int ELEM> struct CheckpointRange {
  static constexpr int kLow = ELEM == kF16 ? 112 : 3;     // 2^-15, 2^-124
  static constexpr int kHigh = ELEM == kF16 ? 135 : 247;  // 2^8, 2^120
};
template <int ELEM> __device__ __forceinline__ int checkpointExponent(float top) {
  const unsigned int bits = __float_as_uint(top);
  const int e = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);  // 448 = 1.75 * 2^8
  return max(CheckpointRange<ELEM>::kLow, min(CheckpointRange<ELEM>::kHigh, e));
}
__device__ __forceinline__ float powerOfExponent(int e) { return __uint_as_float(static_cast<unsigned int>(e) << 23); }
// |v| where v is finite, else 0.
__device__ __forceinline__ float finiteMagnitude(float v) {
  const float a = fabsf(v);
  return a <= 3.402823466e38f ? a : 0.0f;
}
// The multiplication by a power of two is exact (what it pushes below f32's range is far below a code's last bit), so
// the code is rounded once.  Infinities have no code: like NaN they become the format's NaN, so that an overflow is
// still seen behind a checkpoint.
struct CheckpointScale { float inverse, most; };
template <int ELEM> __device__ __forceinline__ CheckpointScale checkpointScale(int e) {
  return {powerOfExponent(254 - e), e == CheckpointRange<ELEM>::kHigh ? 240.0f : 448.0f};
}
__device__ __forceinline__ float scaledForCode(float v, const CheckpointScale &s) {
  const float r = fminf(fmaxf(v * s.inverse, -s.most), s.most);
  return fabsf(v) <= 3.402823466e38f ? r : __uint_as_float(0x7fc00000u);
}
__device__ __forceinline__ unsigned int codePair(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float2 valuePair(unsigned int codes, float power) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes), __NV_E4M3);
  const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
  return make_float2(f.x * power, f.y * power);
}
template <int VEC> __device__ __forceinline__ void valuesOfCodes(const unsigned int (&w)[VEC / 4], float power, float (&v)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC / 4; ++i) {
    const float2 lo = valuePair(w[i] & 0xffffu, power), hi = valuePair(w[i] >> 16, power);
    v[4 * i] = lo.x;
    v[4 * i + 1] = lo.y;
    v[4 * i + 2] = hi.x;
    v[4 * i + 3] = hi.y;
  }
}

// ---- the gate ---------------------------------------------------------------------------------------------------
__device__ __forceinline__ float gateValue(float g, int act) {
  if (act == kActSigmoid) return 1.0f / (1.0f + expf(-g));
  if (act == kActTanh) return tanhf(g);
  return g;
}
// The derivative, from the value.
__device__ __forceinline__ float gateSlope(float a, int act) {
  if (act == kActSigmoid) return a * (1.0f - a);
  if (act == kActTanh) return 1.0f - a * a;
  return 1.0f;
}

} // namespace kernels
} // namespace afir
