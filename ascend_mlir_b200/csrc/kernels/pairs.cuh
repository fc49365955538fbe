// Two f32 values in one 64-bit register: sm_100 adds, multiplies and fuses such pairs in one instruction, which halves
// the arithmetic of row kernels that would otherwise be bound by the number of instructions they issue.
#pragma once

#include "kernels/block_norm_device.cuh"

namespace afir {
namespace kernels {

struct F2 { unsigned long long v; };

__device__ __forceinline__ F2 pairOf(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ F2 splat(float x) { return pairOf(x, x); }
__device__ __forceinline__ float2 valuesOf(F2 a) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(a.v));
  return f;
}
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ float sumOf(F2 a) {
  const float2 f = valuesOf(a);
  return f.x + f.y;
}

// 16 bytes of elements <-> pairs.
template <int ELEM> constexpr int kPairs = ElemOf<ELEM>::kVec / 2;
template <int ELEM> __device__ __forceinline__ void widenPairs(const uint4 &raw, F2 (&p)[kPairs<ELEM>]) {
  const unsigned int w[4] = {raw.x, raw.y, raw.z, raw.w};
  if constexpr (ELEM == kF32) {
    p[0] = pairOf(__uint_as_float(w[0]), __uint_as_float(w[1]));
    p[1] = pairOf(__uint_as_float(w[2]), __uint_as_float(w[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (ELEM == kF16) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        p[i] = pairOf(f.x, f.y);
      } else {
        p[i] = pairOf(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
      }
    }
  }
}
template <int ELEM> __device__ __forceinline__ uint4 narrowPairs(const F2 (&p)[kPairs<ELEM>]) {
  unsigned int w[4];
  if constexpr (ELEM == kF32) {
    const float2 a = valuesOf(p[0]), b = valuesOf(p[1]);
    w[0] = __float_as_uint(a.x);
    w[1] = __float_as_uint(a.y);
    w[2] = __float_as_uint(b.x);
    w[3] = __float_as_uint(b.y);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = valuesOf(p[i]);
      if constexpr (ELEM == kF16) {
        const __half2 h = __floats2half2_rn(f.x, f.y);
        w[i] = *reinterpret_cast<const unsigned int *>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
        w[i] = *reinterpret_cast<const unsigned int *>(&h);
      }
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <int ELEM> __device__ __forceinline__ void loadPairs(const void *p, int64_t at, F2 (&v)[kPairs<ELEM>]) {
  widenPairs<ELEM>(*reinterpret_cast<const uint4 *>(static_cast<const typename ElemOf<ELEM>::Type *>(p) + at), v);
}
template <int ELEM> __device__ __forceinline__ void storePairs(void *p, int64_t at, const F2 (&v)[kPairs<ELEM>]) {
  *reinterpret_cast<uint4 *>(static_cast<typename ElemOf<ELEM>::Type *>(p) + at) = narrowPairs<ELEM>(v);
}
// A parameter vector: of the rows' type or f32 (uniform over the launch); it stays in L1 from row to row.
template <int ELEM> __device__ __forceinline__ void loadParamPairs(const void *p, int type, int at, F2 (&v)[kPairs<ELEM>]) {
  if (ELEM == kF32 || type != kF32) {
    loadPairs<ELEM>(p, at, v);
  } else {
    const float4 *q = reinterpret_cast<const float4 *>(static_cast<const float *>(p) + at);
#pragma unroll
    for (int i = 0; i < kPairs<ELEM> / 2; ++i) {
      const float4 f = q[i];
      v[2 * i] = pairOf(f.x, f.y);
      v[2 * i + 1] = pairOf(f.z, f.w);
    }
  }
}
// The codes of one vector (8 or 4 bytes in the low words of `raw`) times their power.
template <int ELEM> __device__ __forceinline__ void codePairs(const uint2 &raw, int exponent, F2 (&v)[kPairs<ELEM>]) {
  const F2 power = splat(powerOfExponent(exponent));
#pragma unroll
  for (int i = 0; i < kPairs<ELEM>; ++i) {
    const unsigned int w = i < 2 ? raw.x : raw.y;
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>((w >> ((i & 1) * 16)) & 0xffffu), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
    v[i] = pairOf(f.x, f.y) * power;
  }
}
// act(gate) of a vector in place; the derivative from the value.  The row kernels' sigmoid takes the hardware's exponential
// and reciprocal (a few units in the last place of f32, far below a 16-bit step).
template <int N> __device__ __forceinline__ void gatePairs(F2 (&g)[N], int act) {
  if (act == kActNone) return;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float2 f = valuesOf(g[i]);
    if (act == kActSigmoid) g[i] = pairOf(__fdividef(1.0f, 1.0f + __expf(-f.x)), __fdividef(1.0f, 1.0f + __expf(-f.y)));
    else g[i] = pairOf(tanhf(f.x), tanhf(f.y));
  }
}
__device__ __forceinline__ F2 gateSlopePair(F2 a, int act) {
  const F2 one = splat(1.0f), minus = splat(-1.0f);
  if (act == kActSigmoid) return a * fma2(a, minus, one);
  if (act == kActTanh) return fma2(a * minus, a, one);
  return one;
}

// ---- rows fetched ahead -------------------------------------------------------------------------------------------
// Every thread copies the very vectors that it will use into slots of its own in shared memory, asynchronously and
// several rows ahead, so that nothing has to be signalled between threads: waiting for one's own copies is enough.
__device__ __forceinline__ void copyAhead16(void *slot, const void *from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<unsigned int>(__cvta_generic_to_shared(slot))), "l"(from) : "memory");
}
__device__ __forceinline__ void copyAhead8(void *slot, const void *from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(static_cast<unsigned int>(__cvta_generic_to_shared(slot))), "l"(from) : "memory");
}
__device__ __forceinline__ void copyAhead4(void *slot, const void *from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(static_cast<unsigned int>(__cvta_generic_to_shared(slot))), "l"(from) : "memory");
}
__device__ __forceinline__ void copiesCommit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Until all but the newest `left` groups have arrived (left = 1, 2 or 3).
__device__ __forceinline__ void copiesWait(int left) {
  if (left == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else if (left == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else asm volatile("cp.async.wait_group 3;" ::: "memory");
}

} // namespace kernels
} // namespace afir
