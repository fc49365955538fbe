// Two f32 values in one 64-bit register: sm_100 adds, multiplies and fuses such pairs in one instruction, which halves
// the arithmetic of row kernels that would otherwise be bound by the number of instructions they issue.
#pragma once

#include <type_traits>

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
// A parameter vector: of the rows' type or f32 (uniform over the launch).
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
// act(gate) of a vector in place; the derivative from the value.  Of f32 rows as gateValue has it.  In 16-bit rows the sigmoid takes
// CUDA's fast exponential and division, since these kernels are bound by the instructions they issue: with their published
// bounds, (2 + 1.16 |g|) and 2 units in the last place, it is off by less than 4e-7, and by 2.5e-6 of itself down to g = -14,
// where the stored type's half step is 4.9e-4 (f16); beyond |g| = 87 it is 0 or 1, as f32's own to 1e-37.
template <int ELEM> __device__ __forceinline__ float sigmoidOf(float g) {
  if constexpr (ELEM == kF32) return gateValue(g, kActSigmoid);
  else return __fdividef(1.0f, 1.0f + __expf(-g));
}
template <int ELEM> __device__ __forceinline__ void gatePairs(F2 (&g)[kPairs<ELEM>], int act) {
  if (act == kActNone) return;
#pragma unroll
  for (int i = 0; i < kPairs<ELEM>; ++i) {
    const float2 f = valuesOf(g[i]);
    if (act == kActSigmoid) g[i] = pairOf(sigmoidOf<ELEM>(f.x), sigmoidOf<ELEM>(f.y));
    else g[i] = pairOf(tanhf(f.x), tanhf(f.y));
  }
}
// The derivative of the activation from its value, as a polynomial in it: a - a^2 (sigmoid), 1 - a^2 (tanh), 1.
struct GateSlope { F2 c0, c1, c2; };
__device__ __forceinline__ GateSlope gateSlopeOf(int act) {
  return {splat(act == kActSigmoid ? 0.0f : 1.0f), splat(act == kActSigmoid ? 1.0f : 0.0f), splat(act == kActNone ? 0.0f : -1.0f)};
}
__device__ __forceinline__ F2 slopeAt(const GateSlope &g, F2 a) { return fma2(a, fma2(a, g.c2, g.c1), g.c0); }

// ---- packing a vector -----------------------------------------------------------------------------------------------
// Largest magnitude among 16 bytes of elements, NaN left out; 16-bit types compare as they are, two at a time.
template <int ELEM> __device__ __forceinline__ float largestMagnitude(const uint4 &raw) {
  if constexpr (ELEM == kF32) {
    return fmaxf(fmaxf(fabsf(__uint_as_float(raw.x)), fabsf(__uint_as_float(raw.y))), fmaxf(fabsf(__uint_as_float(raw.z)), fabsf(__uint_as_float(raw.w))));
  } else {
    using T2 = typename std::conditional<ELEM == kF16, __half2, __nv_bfloat162>::type;
    const unsigned int w[4] = {raw.x & 0x7fff7fffu, raw.y & 0x7fff7fffu, raw.z & 0x7fff7fffu, raw.w & 0x7fff7fffu};
    const T2 *v = reinterpret_cast<const T2 *>(w);
    const T2 m = __hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3]));
    return fmaxf(ElemOf<ELEM>::widen(m.x), ElemOf<ELEM>::widen(m.y));
  }
}
// A vector's codes: the lanes of a block of 128 columns (128 / VEC neighbours, all lanes of the warp take part) agree on the
// power, whose exponent is returned.  In the ordinary case, no infinity in
// the block and no magnitude that needs the highest power, a code is one product and one conversion: the power brings
// every magnitude to 448 or less.  (f16 multiplies in f16: a product below its normal range is below the smallest code's
// half step as well.)
template <int ELEM> __device__ __forceinline__ int codesOf(const uint4 &raw, unsigned int (&codes)[ElemOf<ELEM>::kVec / 4]) {
  constexpr int VEC = ElemOf<ELEM>::kVec, kGroup = kCheckpointBlock / VEC, W = VEC / 4;
  float top = largestMagnitude<ELEM>(raw);
#pragma unroll
  for (int o = kGroup / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  int e8 = checkpointExponent<ELEM>(top);
  if (!__any_sync(0xffffffffu, e8 == CheckpointRange<ELEM>::kHigh)) {
    const float inverse = powerOfExponent(254 - e8);
    if constexpr (ELEM == kF16) {
      const __half2 scale = __float2half2_rn(inverse);
      const __half2 *v = reinterpret_cast<const __half2 *>(&raw);
      unsigned int q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __half2 r = __hmul2(v[i], scale);
        q[i] = __nv_cvt_halfraw2_to_fp8x2(static_cast<__half2_raw>(r), __NV_SATFINITE, __NV_E4M3);
      }
      codes[0] = q[0] | (q[1] << 16);
      if constexpr (W > 1) codes[W - 1] = q[2] | (q[3] << 16);
    } else {
      F2 v[VEC / 2];
      widenPairs<ELEM>(raw, v);
      const F2 scale = splat(inverse);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float2 lo = valuesOf(v[2 * i] * scale), hi = valuesOf(v[2 * i + 1] * scale);
        codes[i] = codePair(lo.x, lo.y) | (codePair(hi.x, hi.y) << 16);
      }
    }
  } else {
    float v[VEC];
    unpack<ELEM, VEC>(raw, v);
    top = 0.0f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) top = fmaxf(top, finiteMagnitude(v[e]));
#pragma unroll
    for (int o = kGroup / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    e8 = checkpointExponent<ELEM>(top);
    const CheckpointScale s = checkpointScale<ELEM>(e8);
#pragma unroll
    for (int i = 0; i < W; ++i)
      codes[i] = codePair(scaledForCode(v[4 * i], s), scaledForCode(v[4 * i + 1], s)) |
                 (codePair(scaledForCode(v[4 * i + 2], s), scaledForCode(v[4 * i + 3], s)) << 16);
  }
  return e8;
}
template <int ELEM>
__device__ __forceinline__ void packVector(const uint4 &raw, bool live, int col, int64_t row, const CheckpointOut &c) {
  constexpr int W = ElemOf<ELEM>::kVec / 4;
  unsigned int codes[W];
  const int e8 = codesOf<ELEM>(raw, codes);
  if (!live) return;
  uint8_t *to = c.codes + row * c.codesLd + col;
  if constexpr (W == 2) *reinterpret_cast<uint2 *>(to) = make_uint2(codes[0], codes[W - 1]);
  else *reinterpret_cast<unsigned int *>(to) = codes[0];
  if (col % kCheckpointBlock == 0) c.exps[row * c.expsLd + col / kCheckpointBlock] = static_cast<uint8_t>(e8);
}

// ---- rows fetched ahead -------------------------------------------------------------------------------------------
// Every thread copies the very vectors that it will use into slots of its own in shared memory, asynchronously and
// several rows ahead, so that nothing has to be signalled between threads: waiting for one's own copies is enough.
__device__ __forceinline__ void copyAhead16(unsigned int slot, const void *from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slot), "l"(from) : "memory");
}
__device__ __forceinline__ void copyAhead8(unsigned int slot, const void *from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(slot), "l"(from) : "memory");
}
__device__ __forceinline__ void copyAhead4(unsigned int slot, const void *from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(slot), "l"(from) : "memory");
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
