// A ring of buffers that is filled round by round, each buffer with an mbarrier that completes one phase per round.
#pragma once

#ifdef __CUDACC__
#define AFIR_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define AFIR_HOST_DEVICE inline
#endif

namespace afir {
namespace kernels {

// Place in a ring of N and the parity of its round.
template <int N> struct Ring {
  int at = 0;
  unsigned int phase = 0;
  AFIR_HOST_DEVICE void next() {
    if (++at == N) {
      at = 0;
      phase ^= 1u;
    }
  }
};

// Before the next fill, which goes to place `at` of a round of parity `phase`: the parity to wait for until the newest fill of
// place s is complete.  Of a place that was never filled it is the one that a fresh barrier answers at once.  (Whichever the
// barrier's state, one of the two parities is answered at once: waiting for either is no wait.)
AFIR_HOST_DEVICE unsigned int newestFillParity(int s, int at, unsigned int phase) { return s < at ? phase : phase ^ 1u; }

} // namespace kernels
} // namespace afir
