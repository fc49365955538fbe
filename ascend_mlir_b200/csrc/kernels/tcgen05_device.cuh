// Pieces shared by the tensor-core kernels (matmul_tcgen05.cu, checkpoint_grad_tcgen05.cu): mbarrier waits with a limit, TMA
// loads, tcgen05 instructions, and the host side of tensor maps.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <mutex>

#include "kernels/kernels.h"
#include "kernels/ring.h"

namespace afir {
namespace kernels {

constexpr unsigned long long kWaitLimitNs = 2000000000ull;

// Per-CTA abort state in shared memory: raised by the first wait that runs out, seen by every role's next check.
struct AbortState {
  int flag;
  unsigned int *status;  // where the time-out is reported
};

// ---- PTX wrappers ------------------------------------------------------------------------------
__device__ __forceinline__ unsigned int smemAddr(const void *p) {
  return static_cast<unsigned int>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ unsigned long long globalTimerNs() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ void mbarInit(unsigned int bar, unsigned int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbarExpectTx(unsigned int bar, unsigned int bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbarArrive(unsigned int bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbarTryWait(unsigned int bar, unsigned int parity) {
  unsigned int done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}
// Bounded wait.  Returns false when the abort flag is (or becomes) raised.
__device__ __forceinline__ bool mbarWait(unsigned int bar, unsigned int parity, volatile AbortState *abortFlag, unsigned int role) {
  if (mbarTryWait(bar, parity)) return true;
  const unsigned long long t0 = globalTimerNs();
  unsigned int spins = 0;
  while (true) {
    if (mbarTryWait(bar, parity)) return true;
    // epilogue warps wait a whole mainloop for their accumulator: back off instead of burning issue slots and power
    if (role == 2) __nanosleep(256);
    else if (role == 0) __nanosleep(64);  // the producer is normally a full ring ahead: poll lazily
    if ((++spins & 63u) == 0) {
      if (abortFlag->flag) return false;
      if (globalTimerNs() - t0 > kWaitLimitNs) {
        abortFlag->flag = 1;
        atomicCAS(abortFlag->status, 0u, (1u << 8) | role);
        return false;
      }
    }
  }
}
// Waits for a phase, 1 ms at most: for copies into, or products that read, memory that a CTA is about to give up.
__device__ __forceinline__ void mbarDrain(unsigned int bar, unsigned int parity) {
  const unsigned long long t0 = globalTimerNs();
  while (!mbarTryWait(bar, parity) && globalTimerNs() - t0 < 1000000ull) {
  }
}
__device__ __forceinline__ void tmaLoad2d(unsigned int dst, const CUtensorMap *map, int x, int y, unsigned int bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void prefetchTensorMap(const CUtensorMap *map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
__device__ __forceinline__ void tcgen05FenceBefore() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tcgen05FenceAfter() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmemAlloc(unsigned int dstSmem, unsigned int cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dstSmem), "r"(cols) : "memory");
}
__device__ __forceinline__ void tmemRelinquish() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmemDealloc(unsigned int taddr, unsigned int cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
__device__ __forceinline__ void ummaF16(unsigned int dTmem, unsigned long long aDesc, unsigned long long bDesc,
                                        unsigned int idesc, unsigned int accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(dTmem), "l"(aDesc), "l"(bDesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives on `bar` once every tcgen05.mma issued so far by this thread has completed.
__device__ __forceinline__ void ummaCommit(unsigned int bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmemLoad32(unsigned int taddr, unsigned int (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmemLoadWait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Shared-memory matrix descriptor (tcgen05): start address, leading/stride byte offsets (>>4),
// descriptor version 1, 128-byte swizzle.
__device__ __forceinline__ unsigned long long smemDesc(unsigned int addr, unsigned int lboBytes, unsigned int sboBytes) {
  unsigned long long d = 0;
  d |= static_cast<unsigned long long>((addr & 0x3FFFFu) >> 4);
  d |= static_cast<unsigned long long>((lboBytes >> 4) & 0x3FFFu) << 16;
  d |= static_cast<unsigned long long>((sboBytes >> 4) & 0x3FFFu) << 32;
  d |= 1ull << 46;  // descriptor version (Blackwell)
  d |= 2ull << 61;  // SWIZZLE_128B
  return d;
}

// Eight f32 results -> 16-byte pieces of the output row (two pieces for f32, one for 16-bit types).
template <int OUT> struct OutPack;
template <> struct OutPack<kF32> {
  static constexpr int kBytes = 4;
  static constexpr int kPieces = 2;
  __device__ __forceinline__ static void pack8(const float *v, uint4 *q) {
    q[0] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    q[1] = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
  }
};
template <> struct OutPack<kBF16> {
  static constexpr int kBytes = 2;
  static constexpr int kPieces = 1;
  __device__ __forceinline__ static void pack8(const float *v, uint4 *q) {
    __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
    __nv_bfloat162 c = __floats2bfloat162_rn(v[4], v[5]), d = __floats2bfloat162_rn(v[6], v[7]);
    q[0] = make_uint4(*reinterpret_cast<unsigned int *>(&a), *reinterpret_cast<unsigned int *>(&b),
                      *reinterpret_cast<unsigned int *>(&c), *reinterpret_cast<unsigned int *>(&d));
  }
};
template <> struct OutPack<kF16> {
  static constexpr int kBytes = 2;
  static constexpr int kPieces = 1;
  __device__ __forceinline__ static void pack8(const float *v, uint4 *q) {
    __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
    __half2 c = __floats2half2_rn(v[4], v[5]), d = __floats2half2_rn(v[6], v[7]);
    q[0] = make_uint4(*reinterpret_cast<unsigned int *>(&a), *reinterpret_cast<unsigned int *>(&b),
                      *reinterpret_cast<unsigned int *>(&c), *reinterpret_cast<unsigned int *>(&d));
  }
};

// ---- host side ----------------------------------------------------------------------------------------------
using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                   const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encodeTiled() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

inline bool makeMap2d(CUtensorMap *map, CUtensorMapDataType type, const void *base, uint64_t inner, uint64_t outer,
               uint64_t rowBytes, uint32_t boxInner, uint32_t boxOuter,
                      CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
  EncodeTiledFn fn = encodeTiled();
  if (!fn) return false;
  cuuint64_t dims[2] = {inner, outer};
  cuuint64_t strides[1] = {rowBytes};
  cuuint32_t box[2] = {boxInner, boxOuter};
  cuuint32_t elemStrides[2] = {1, 1};
  return fn(map, type, 2, const_cast<void *>(base), dims, strides, box, elemStrides, CU_TENSOR_MAP_INTERLEAVE_NONE,
            swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A function attribute belongs to the function ON THE CURRENT DEVICE: a process that runs the matmul on several
// GPUs has to set it once on each of them.  `run` calls `set` the first time it is reached with a given device
// current (and again after a failure) and returns that device's result.
struct PerDeviceOnce {
  std::mutex mu;
  bool done[64] = {false};
  template <class F> cudaError_t run(F set) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    if (device < 0 || device >= 64) return set();
    std::lock_guard<std::mutex> lock(mu);
    if (done[device]) return cudaSuccess;
    e = set();
    done[device] = e == cudaSuccess;
    return e;
  }
};

} // namespace kernels
} // namespace afir
