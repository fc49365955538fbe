// Vectors of rows that do not start on 16 bytes, or end inside a vector (odd widths, odd slices).
//
// A thread still owns 16 bytes' worth of neighbouring columns.  It reads the two aligned pieces that hold them and shifts (the
// shift is the same for a whole row), which costs a dozen instructions instead of a load per element, and writes in pieces
// of 4 bytes.  An aligned piece may reach up to 15 bytes beyond the row, into the row before or behind it: never
// beyond the tensor, since the first and the last row, and rows shorter than 32 bytes, are read by elements.
#pragma once

#include "kernels/pairs.cuh"

namespace afir {
namespace kernels {

// Whether row `row` of `rows` may be read in aligned pieces.
__device__ __forceinline__ bool innerRow(int64_t row, int64_t rows, int64_t rowBytes) { return row > 0 && row + 1 < rows && rowBytes >= 32; }

// The 16 bytes at `p` (which is aligned to its elements).
__device__ __forceinline__ uint4 shiftedLoad16(const char *p) {
  const unsigned int m = static_cast<unsigned int>(reinterpret_cast<uintptr_t>(p)) & 15u;
  const uint4 *q = reinterpret_cast<const uint4 *>(p - m);
  const uint4 lo = q[0];
  if (m == 0) return lo;
  const uint4 hi = q[1];
  const unsigned int r[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  unsigned int a[6], b[5];
#pragma unroll
  for (int i = 0; i < 6; ++i) a[i] = (m & 8u) ? r[i + 2] : r[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) b[i] = (m & 4u) ? a[i + 1] : a[i];
  const unsigned int bits = (m & 3u) * 8u;
  return make_uint4(__funnelshift_r(b[0], b[1], bits), __funnelshift_r(b[1], b[2], bits), __funnelshift_r(b[2], b[3], bits), __funnelshift_r(b[3], b[4], bits));
}
// The 8 or 4 bytes at `p`, in the low words.
template <int BYTES> __device__ __forceinline__ uint2 shiftedLoadCodes(const uint8_t *p) {
  const unsigned int m = static_cast<unsigned int>(reinterpret_cast<uintptr_t>(p)) & 3u;
  const unsigned int *q = reinterpret_cast<const unsigned int *>(p - m);
  uint2 v = make_uint2(q[0], BYTES == 8 ? q[1] : 0u);
  if (m != 0) {
    const unsigned int last = q[BYTES / 4], bits = m * 8u;
    v = BYTES == 8 ? make_uint2(__funnelshift_r(v.x, v.y, bits), __funnelshift_r(v.y, last, bits)) : make_uint2(__funnelshift_r(v.x, last, bits), 0u);
  }
  return v;
}

// The vector of columns [col, col + VEC) of the row that begins at element `rowAt`; zeros from `cols` on.
template <int ELEM, int VEC>
__device__ __forceinline__ void looseLoad(const void *base, int64_t rowAt, int col, int cols, bool inner, float (&v)[VEC]) {
  using T = typename ElemOf<ELEM>::Type;
  const T *p = static_cast<const T *>(base) + rowAt + col;
  if (inner && col + VEC <= cols) {
    unpack<ELEM, VEC>(shiftedLoad16(reinterpret_cast<const char *>(p)), v);
    return;
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) v[e] = col + e < cols ? ElemOf<ELEM>::widen(p[e]) : 0.0f;
}
template <int ELEM, int VEC> __device__ __forceinline__ void looseStore(void *base, int64_t rowAt, int col, int cols, const float (&v)[VEC]) {
  using T = typename ElemOf<ELEM>::Type;
  T *p = static_cast<T *>(base) + rowAt + col;
  if (col + VEC <= cols) {
    const uint4 q = pack<ELEM, VEC>(v);
    const unsigned int m = static_cast<unsigned int>(reinterpret_cast<uintptr_t>(p)) & 15u;
    if (m == 0) {
      *reinterpret_cast<uint4 *>(p) = q;
    } else if ((m & 3u) == 0) {
      unsigned int *w = reinterpret_cast<unsigned int *>(p);
      w[0] = q.x;
      w[1] = q.y;
      w[2] = q.z;
      w[3] = q.w;
    } else {  // 16-bit elements, two bytes off a word
      unsigned short *h = reinterpret_cast<unsigned short *>(p);
      unsigned int *w = reinterpret_cast<unsigned int *>(h + 1);
      h[0] = static_cast<unsigned short>(q.x);
      w[0] = __funnelshift_r(q.x, q.y, 16);
      w[1] = __funnelshift_r(q.y, q.z, 16);
      w[2] = __funnelshift_r(q.z, q.w, 16);
      h[7] = static_cast<unsigned short>(q.w >> 16);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e)
    if (col + e < cols) p[e] = ElemOf<ELEM>::narrow(v[e]);
}
// A parameter vector's part; zeros from `cols` on.
template <int ELEM, int VEC> __device__ __forceinline__ void looseParam(const void *p, int type, int col, int cols, float (&v)[VEC]) {
  if (col + VEC <= cols && (reinterpret_cast<uintptr_t>(p) & 15u) == 0) {
    loadParam<ELEM, VEC>(p, type, col, v);
    return;
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    float one[1] = {0.0f};
    if (col + e < cols) loadParam<ELEM, 1>(p, type, col + e, one);
    v[e] = one[0];
  }
}
template <int VEC> __device__ __forceinline__ void looseCheckpoint(const CheckpointIn &c, int64_t row, int col, int cols, bool inner, float (&v)[VEC]) {
  const float power = powerOfExponent(c.exps[row * c.expsLd + col / kCheckpointBlock]);
  const uint8_t *p = c.codes + row * c.codesLd + col;
  unsigned int w[VEC / 4];
  if (inner && col + VEC <= cols) {
    const uint2 r = shiftedLoadCodes<VEC>(p);
    w[0] = r.x;
    if constexpr (VEC == 8) w[1] = r.y;
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      w[i] = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + 4 * i + e < cols) w[i] |= static_cast<unsigned int>(p[4 * i + e]) << (8 * e);
    }
  }
  valuesOfCodes<VEC>(w, power, v);
}
// Codes of a vector into [col, col + 4*W) of a row, as far as `cols`.
template <int W> __device__ __forceinline__ void looseCodes(uint8_t *p, int col, int cols, const unsigned int (&codes)[W]) {
  const unsigned int m = static_cast<unsigned int>(reinterpret_cast<uintptr_t>(p)) & 3u;
  if (col + 4 * W <= cols && m == 0) {
#pragma unroll
    for (int i = 0; i < W; ++i) reinterpret_cast<unsigned int *>(p)[i] = codes[i];
  } else if (col + 4 * W <= cols && m == 2) {
#pragma unroll
    for (int i = 0; i < 2 * W; ++i) reinterpret_cast<unsigned short *>(p)[i] = static_cast<unsigned short>(codes[i >> 1] >> ((i & 1) * 16));
  } else {
#pragma unroll
    for (int i = 0; i < 4 * W; ++i)
      if (col + i < cols) p[i] = static_cast<uint8_t>(codes[i >> 2] >> ((i & 3) * 8));
  }
}
template <int VEC> __device__ __forceinline__ void looseSums(float *to, int col, int cols, const float (&v)[VEC]) {
#pragma unroll
  for (int e = 0; e < VEC; ++e)
    if (col + e < cols) to[e] = v[e];
}

} // namespace kernels
} // namespace afir
