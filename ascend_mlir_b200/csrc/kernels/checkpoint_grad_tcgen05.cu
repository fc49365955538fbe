// Weight gradient from an 8-bit checkpoint, for sm_100a:
//     dweight[D, N] = restore(codes, exps)[T, D]^T . dy[T, N]
// The restored activation never exists in HBM: codes come in as they are (one byte per element), are widened in the SM to the
// 16-bit type of dy, which is exact (four significant bits times a power of two), and go to the tensor cores from shared
// memory.
//
//   warp 0      TMA producer of dy: [64 tokens x 256] per stage;
//   warp 1      MMA issuer: tcgen05.mma.cta_group::1.kind::f16, 128 x 256 x 16, both operands with their long side
//               contiguous (tokens are the summed dimension and the rows of both tensors);
//   warps 2..17 load codes straight into registers two stages ahead (a token's 128 columns are one line), convert them into
//               the A operand (128-byte swizzle), and write the finished tile out: tcgen05.ld, convert, 16-byte
//               stores that cover whole 128-byte lines.
// What bounds it is shared memory: a stage of 256 x 256 x 64 takes 1024 cycles of the tensor cores, which read 96 KB of
// operands (768 cycles) while dy comes in (256) and A is written (256).  Codes staged in shared memory as well cost another
// 256 cycles and were measured slower.
// Measured, 8192^3 bf16: 844 to 860 us alone (1.28 to 1.30 PFLOP/s, tensor pipe active 70 % of the time), 935 in a loop of
// seconds under the power limit; a library product of two 16-bit tensors takes 664 and 728 there.  300 x 1024 x 1024 f16: 8.2 us, most
// of it start-up and one tile's way through the pipeline.
// The tensor cores cut their f32 sums off toward zero: over 8192 tokens in one slice the result is off by 3.6e-6 of itself (2-norm),
// rounded sums by 3.6e-7; what is read has four significant bits.
// TM = 128 * MB rows of dweight per CTA; MB = 2 halves what dy costs per flop.  One persistent CTA per SM.  Where the
// tiles of dweight are fewer than the SMs the tokens are cut into slices whose partial tiles (f32) a second kernel adds in order.
//
// Every wait on an mbarrier is bounded, as in matmul_tcgen05.cu: after about 2 s the launch's status word is set, every role leaves
// its loop, copies in flight are waited for (bounded), tensor memory is freed and the kernel returns.
#include <algorithm>
#include <cstdio>

#include "kernels/block_norm.h"
#include "kernels/block_norm_device.cuh"
#include "kernels/launch_util.h"
#include "kernels/pairs.cuh"
#include "kernels/tcgen05_device.cuh"

namespace afir {
namespace kernels {
namespace {

// 0, or (1 << 8) | the role whose wait ran out first.
__device__ unsigned int checkpointGradStatusWords[kCheckpointGradStatusWords];

constexpr int kTileN = 256;
constexpr int kTokens = 64;                      // summed per stage
constexpr int kBlockBytes = kTokens * 64 * 2;    // 64 tokens x 64 columns of a 16-bit operand
constexpr int kBStage = 4 * kBlockBytes;
constexpr int kConvertWarps = 16;
constexpr int kThreads = 64 + 32 * kConvertWarps;

template <int MB> struct GradShape {
  static constexpr int kTileM = 128 * MB;
  static constexpr int kATileBytes = MB * 2 * kBlockBytes;
  static constexpr int kBStages = 4, kATiles = MB == 1 ? 4 : 3;
  static constexpr int kTmemCols = MB * kTileN;
  static constexpr size_t kAAt = static_cast<size_t>(kBStages) * kBStage, kControlAt = kAAt + static_cast<size_t>(kATiles) * kATileBytes;
  static_assert(kATiles * kATileBytes >= kConvertWarps * 4096, "the A tiles double as the staging area of the output");
};
template <int MB> struct GradControl {
  using S = GradShape<MB>;
  unsigned long long bFull[S::kBStages], bEmpty[S::kBStages], aFull[S::kATiles], aEmpty[S::kATiles];
  unsigned long long tileFull, tileEmpty, drained;
  unsigned int tmemBase;
  AbortState abort;
};
template <int MB> constexpr size_t gradSmemBytes() { return 1024 + GradShape<MB>::kControlAt + sizeof(GradControl<MB>); }
static_assert(gradSmemBytes<1>() <= 227 * 1024 && gradSmemBytes<2>() <= 227 * 1024, "shared memory of a CTA");

struct GradParams {
  int D, N, T;
  int tilesM, tilesN, kBlocks, splits, kPerSplit, band;
  const uint8_t *codes, *exps;
  int64_t codesLd, expsLd;
  void *out;       // dweight, or the partial tiles [splits][D][N] f32
  int64_t outLd;
  int64_t splitStride;
  int accumulate;
  unsigned int idesc;
  int statusWord;
};

// 16 codes -> 16 values of the operand type, times the power (2^k as f32 bits).
template <int ELEM> __device__ __forceinline__ void widenCodes(const uint4 &raw, float power, uint4 (&out)[2]) {
  const unsigned int w[4] = {raw.x, raw.y, raw.z, raw.w};
  unsigned int r[8];
  if constexpr (ELEM == kF16) {
    // the power as f16: 2^-15 (a subnormal) to 2^8, exact, and so is the product
    const __half2 scale = __float2half2_rn(power);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>((w[i >> 1] >> ((i & 1) * 16)) & 0xffffu), __NV_E4M3);
      const __half2 m = __hmul2(*reinterpret_cast<const __half2 *>(&h), scale);
      r[i] = *reinterpret_cast<const unsigned int *>(&m);
    }
  } else {
    const F2 scale = splat(power);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>((w[i >> 1] >> ((i & 1) * 16)) & 0xffffu), __NV_E4M3);
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
      const float2 m = valuesOf(pairOf(f.x, f.y) * scale);
      const __nv_bfloat162 b = __floats2bfloat162_rn(m.x, m.y);
      r[i] = *reinterpret_cast<const unsigned int *>(&b);
    }
  }
  out[0] = make_uint4(r[0], r[1], r[2], r[3]);
  out[1] = make_uint4(r[4], r[5], r[6], r[7]);
}

// 16 bytes that nobody in this SM reads again soon.
__device__ __forceinline__ uint4 loadOnce16(const uint8_t *p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

__device__ __forceinline__ uint4 addF32(const uint4 &a, const uint4 &b) {
  return make_uint4(__float_as_uint(__uint_as_float(a.x) + __uint_as_float(b.x)), __float_as_uint(__uint_as_float(a.y) + __uint_as_float(b.y)),
                    __float_as_uint(__uint_as_float(a.z) + __uint_as_float(b.z)), __float_as_uint(__uint_as_float(a.w) + __uint_as_float(b.w)));
}

template <int ELEM, int OUT, int MB>
__global__ void __launch_bounds__(kThreads, 1)
checkpointGradKernel(const __grid_constant__ CUtensorMap mapDy, const __grid_constant__ GradParams prm) {
  using S = GradShape<MB>;
  constexpr int kBStages = S::kBStages, kATiles = S::kATiles;
  extern __shared__ unsigned char smemRaw[];
  unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smemRaw) + 1023) & ~uintptr_t(1023));
  unsigned char *aTiles = smem + S::kAAt;
  GradControl<MB> *ctl = reinterpret_cast<GradControl<MB> *>(smem + S::kControlAt);
  volatile AbortState *abortFlag = &ctl->abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = prm.tilesM * prm.tilesN, units = tiles * prm.splits;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kBStages; ++s) {
      mbarInit(smemAddr(&ctl->bFull[s]), 1);
      mbarInit(smemAddr(&ctl->bEmpty[s]), 1);
    }
    for (int a = 0; a < kATiles; ++a) {
      mbarInit(smemAddr(&ctl->aFull[a]), kConvertWarps);
      mbarInit(smemAddr(&ctl->aEmpty[a]), 1);
    }
    mbarInit(smemAddr(&ctl->tileFull), 1);
    mbarInit(smemAddr(&ctl->drained), 1);
    mbarInit(smemAddr(&ctl->tileEmpty), kConvertWarps);
    ctl->abort.flag = 0;
    ctl->abort.status = &checkpointGradStatusWords[prm.statusWord];
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    prefetchTensorMap(&mapDy);
  }
  if (warp == 1) {
    tmemAlloc(smemAddr(&ctl->tmemBase), S::kTmemCols);
    tmemRelinquish();
  }
  tcgen05FenceBefore();
  __syncthreads();
  tcgen05FenceAfter();
  const unsigned int tmemBase = ctl->tmemBase;

  // Slices outermost; inside, bands of tile-rows with the rows fastest, so that CTAs running together share operands in L2.
  auto unitCoords = [&](int u, int &tm, int &tn, int &k0, int &k1, int &split) {
    split = u / tiles;
    const int t = u - split * tiles;
    const int bandTiles = prm.band * prm.tilesN;
    const int band = t / bandTiles, within = t - band * bandTiles;
    const int rowsInBand = min(prm.band, prm.tilesM - band * prm.band);
    tm = band * prm.band + within % rowsInBand;
    tn = within / rowsInBand;
    k0 = split * prm.kPerSplit;
    k1 = min(prm.kBlocks, k0 + prm.kPerSplit);
  };

  Ring<kBStages> ring;  // of dy's stages, the producer's
  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
        int tm, tn, k0, k1, split;
        unitCoords(u, tm, tn, k0, k1, split);
        for (int kb = k0; kb < k1; ++kb, ring.next()) {
          if (!mbarWait(smemAddr(&ctl->bEmpty[ring.at]), ring.phase ^ 1u, abortFlag, 0)) { ok = false; break; }
          const unsigned int full = smemAddr(&ctl->bFull[ring.at]), to = smemAddr(smem + static_cast<size_t>(ring.at) * kBStage);
          mbarExpectTx(full, kBStage);
#pragma unroll
          for (int j = 0; j < 4; ++j) tmaLoad2d(to + j * kBlockBytes, &mapDy, tn * kTileN + j * 64, kb * kTokens, full);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      unsigned int unit = 0;
      Ring<kBStages> bRing;
      Ring<kATiles> aRing;
      bool ok = true;
      for (int u = blockIdx.x; u < units && ok; u += gridDim.x, ++unit) {
        int tm, tn, k0, k1, split;
        unitCoords(u, tm, tn, k0, k1, split);
        if (!mbarWait(smemAddr(&ctl->tileEmpty), (unit & 1u) ^ 1u, abortFlag, 1)) break;
        tcgen05FenceAfter();
        for (int kb = k0; kb < k1; ++kb, bRing.next(), aRing.next()) {
          const int s = bRing.at, a = aRing.at;
          // dy's copy and the converted codes: each is waited for where it becomes visible to the tensor cores
          if (!mbarWait(smemAddr(&ctl->bFull[s]), bRing.phase, abortFlag, 1) ||
              !mbarWait(smemAddr(&ctl->aFull[a]), aRing.phase, abortFlag, 1)) { ok = false; break; }
          tcgen05FenceAfter();
          const unsigned int aBase = smemAddr(aTiles + a * S::kATileBytes);
          const unsigned int bBase = smemAddr(smem + static_cast<size_t>(s) * kBStage);
#pragma unroll
          for (int h = 0; h < MB; ++h) {
            const unsigned int dTmem = tmemBase + static_cast<unsigned int>(h * kTileN);
#pragma unroll
            for (int k = 0; k < kTokens / 16; ++k) {
              // 64-column blocks 8192 bytes apart (leading), groups of 8 tokens 1024 bytes apart (stride)
              const unsigned long long aDesc = smemDesc(aBase + h * 2 * kBlockBytes + k * (16 * 128), kBlockBytes, 1024);
              const unsigned long long bDesc = smemDesc(bBase + k * (16 * 128), kBlockBytes, 1024);
              ummaF16(dTmem, aDesc, bDesc, prm.idesc, (kb > k0 || k > 0) ? 1u : 0u);
            }
          }
          ummaCommit(smemAddr(&ctl->bEmpty[s]));
          ummaCommit(smemAddr(&ctl->aEmpty[a]));
        }
        if (!ok) break;
        ummaCommit(smemAddr(&ctl->tileFull));
      }
    }
  } else {
    const int cw = warp - 2;
    constexpr int kSteps = MB * (kTokens / 4) / kConvertWarps;  // 4 tokens x 128 columns per warp and step
    const int half = MB == 2 ? cw & 1 : 0;                      // which 128 columns of the tile
    const int tokenBase = (MB == 2 ? cw >> 1 : cw) * (kSteps * 4) + (lane >> 3);
    const int piece = lane & 7;                                 // 16 columns of the 128
    const int quarter = warp & 3;
    // Eight lanes write one token's 128 columns, two 64-column blocks: those of the second block write their upper half
    // first, so that the eight 16-byte pieces of each store fall on different banks.
    const bool upperFirst = (piece >> 2) != 0;
    int to[kSteps];
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
      const int token = tokenBase + j * 4;
      to[j] = (half * 2 + (piece >> 2)) * kBlockBytes + token * 128 + ((((piece & 3) * 2 + (upperFirst ? 1 : 0)) ^ (token & 7)) << 4);
    }
    unsigned int unit = 0;
    Ring<kATiles> aRing;
    bool ok = true;
    for (int u = blockIdx.x; u < units && ok; u += gridDim.x, ++unit) {
      int tm, tn, k0, k1, split;
      unitCoords(u, tm, tn, k0, k1, split);
      // This thread's codes and their exponents, two stages ahead.  Beyond the last token or column: zeros.
      const int col = tm * S::kTileM + half * 128 + piece * 16;
      const bool colLive = col < prm.D;  // D is a multiple of 16: a piece is wholly inside or outside
      const int64_t firstToken = static_cast<int64_t>(k0) * kTokens + tokenBase;
      const uint8_t *codeRow = prm.codes + firstToken * prm.codesLd + col, *expRow = prm.exps + firstToken * prm.expsLd + tm * MB + half;
      int tokensLeft = prm.T - static_cast<int>(firstToken);
      struct Ahead { uint4 raw[kSteps]; unsigned int exps[kSteps]; };
      auto load = [&](Ahead &a) {
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
          const bool some = colLive && j * 4 < tokensLeft;
          a.raw[j] = make_uint4(0u, 0u, 0u, 0u);
          a.exps[j] = 127u;
          if (some) {
            a.raw[j] = loadOnce16(codeRow + j * 4 * prm.codesLd);
            a.exps[j] = __ldg(expRow + j * 4 * prm.expsLd);
          }
        }
        codeRow += kTokens * prm.codesLd;
        expRow += kTokens * prm.expsLd;
        tokensLeft -= kTokens;
      };
      Ahead now, next, after;
      load(now);
      load(next);
      for (int kb = k0; kb < k1; ++kb, aRing.next()) {
        load(after);
        const int a = aRing.at;
        if (!__all_sync(0xffffffffu, mbarWait(smemAddr(&ctl->aEmpty[a]), aRing.phase ^ 1u, abortFlag, 3))) { ok = false; break; }
        unsigned char *tile = aTiles + a * S::kATileBytes;
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
          uint4 v[2];
          widenCodes<ELEM>(now.raw[j], powerOfExponent(static_cast<int>(now.exps[j])), v);
          *reinterpret_cast<uint4 *>(tile + to[j]) = upperFirst ? v[1] : v[0];
          *reinterpret_cast<uint4 *>(tile + (to[j] ^ 16)) = upperFirst ? v[0] : v[1];
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbarArrive(smemAddr(&ctl->aFull[a]));
        now = next;
        next = after;
      }
      if (!ok) break;

      // ---- the finished tile: four warps share the tensor memory's lanes; for MB = 2 half of the fours take each accumulator
      // and share its columns, for MB = 1 all share the columns.  The A tiles are free (every MMA has completed) and serve as
      // staging.
      if (!__all_sync(0xffffffffu, mbarWait(smemAddr(&ctl->tileFull), unit & 1u, abortFlag, 2))) break;
      tcgen05FenceAfter();
      unsigned char *stg = aTiles + cw * 4096;
      const int share = cw >> 2;
      constexpr int kPerTile = kConvertWarps / 4 / MB, kCols = kTileN / kPerTile;
      const int rowBase = tm * S::kTileM + share / kPerTile * 128 + quarter * 32;
      const int colBegin = share % kPerTile * kCols, colEnd = colBegin + kCols;
      const unsigned int taddr = tmemBase + static_cast<unsigned int>(share / kPerTile * kTileN) + (static_cast<unsigned int>(quarter * 32) << 16);
      constexpr int kColsPerSlice = 128 / OutPack<OUT>::kBytes;
      unsigned char *out = static_cast<unsigned char *>(prm.out) + static_cast<size_t>(split) * prm.splitStride * OutPack<OUT>::kBytes;
#pragma unroll 1
      for (int c = colBegin; c < colEnd; c += kColsPerSlice) {
        if (tn * kTileN + c >= prm.N) break;
#pragma unroll
        for (int part = 0; part < kColsPerSlice / 32; ++part) {
          unsigned int r[32];
          tmemLoad32(taddr + c + part * 32, r);
          tmemLoadWait();
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(r[j * 8 + e]);
            uint4 q[OutPack<OUT>::kPieces];
            OutPack<OUT>::pack8(v, q);
#pragma unroll
            for (int p = 0; p < OutPack<OUT>::kPieces; ++p) {
              const int at = (part * 4 + j) * OutPack<OUT>::kPieces + p;
              *reinterpret_cast<uint4 *>(stg + lane * 128 + ((at ^ (lane & 7)) << 4)) = q[p];
            }
          }
        }
        __syncwarp();
        const int col = tn * kTileN + c + piece * (16 / OutPack<OUT>::kBytes);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int rr = i * 4 + (lane >> 3), row = rowBase + rr;
          uint4 val = *reinterpret_cast<const uint4 *>(stg + rr * 128 + ((piece ^ (rr & 7)) << 4));
          if (row < prm.D && col < prm.N) {  // N is a multiple of 8: a 16-byte piece is wholly inside or outside
            uint4 *to = reinterpret_cast<uint4 *>(out + (static_cast<size_t>(row) * prm.outLd + col) * OutPack<OUT>::kBytes);
            if constexpr (OUT == kF32) {
              if (prm.accumulate) val = addF32(*to, val);
            }
            *to = val;
          }
        }
        __syncwarp();
      }
      tcgen05FenceBefore();
      __syncwarp();
      if (lane == 0) mbarArrive(smemAddr(&ctl->tileEmpty));
      // nobody converts into the A tiles while another warp still reads its staging there
      if (!__all_sync(0xffffffffu, mbarWait(smemAddr(&ctl->tileEmpty), unit & 1u, abortFlag, 3))) break;
    }
  }

  tcgen05FenceBefore();
  __syncthreads();
  // Where a wait ran out, copies may still land in this CTA's shared memory and products read it: they get time to end.
  const bool gaveUp = abortFlag->flag != 0;
  if (gaveUp && threadIdx.x == 0) {
    for (int s = 0; s < kBStages; ++s) mbarDrain(smemAddr(&ctl->bFull[s]), newestFillParity(s, ring.at, ring.phase));
  }
  if (warp == 1) {
    if (gaveUp && lane == 0) {
      ummaCommit(smemAddr(&ctl->drained));
      mbarDrain(smemAddr(&ctl->drained), 0);
    }
    __syncwarp();
    tcgen05FenceAfter();
    tmemDealloc(tmemBase, S::kTmemCols);
  }
}

// The slices' partial tiles, added in slice order; 4 columns per thread.
template <int OUT>
__global__ void __launch_bounds__(256) checkpointGradJoinKernel(const float *partial, int splits, int64_t rows, int cols, void *out, int64_t outLd, int accumulate) {
  const int64_t perRow = cols / 4;
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; u < rows * perRow; u += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = u / perRow;
    const int col = static_cast<int>(u - row * perRow) * 4;
    float4 sum = *reinterpret_cast<const float4 *>(partial + row * cols + col);
    for (int s = 1; s < splits; ++s) {
      const float4 f = *reinterpret_cast<const float4 *>(partial + (s * rows + row) * cols + col);
      sum.x += f.x;
      sum.y += f.y;
      sum.z += f.z;
      sum.w += f.w;
    }
    if constexpr (OUT == kF32) {
      float4 *to = reinterpret_cast<float4 *>(static_cast<float *>(out) + row * outLd + col);
      if (accumulate) {
        const float4 f = *to;
        sum = make_float4(sum.x + f.x, sum.y + f.y, sum.z + f.z, sum.w + f.w);
      }
      *to = sum;
    } else {
      const float v[8] = {sum.x, sum.y, sum.z, sum.w, 0.f, 0.f, 0.f, 0.f};
      uint4 q[1];
      OutPack<OUT>::pack8(v, q);
      *reinterpret_cast<uint2 *>(static_cast<unsigned short *>(out) + row * outLd + col) = make_uint2(q[0].x, q[0].y);
    }
  }
}

struct SplitPlan { int mb, tilesM, tilesN, kBlocks, splits, kPerSplit; };

// 256-row tiles where they keep at least half of the SMs busy (each moves half of dy's bytes per flop; 8192 x 2048 x 4096:
// 119 us, 153 in 128-row tiles, and both 79 at 2048 x 2048, below the bound), else 128-row tiles; tokens cut into slices where the
// tiles leave SMs idle and a slice still has work for its ring (1024 x 1024: 8192 tokens 36 us, 72 uncut; 2048 tokens 23.5 and
// 24.6; 300 tokens in two slices 19.5, uncut 12.3).
SplitPlan splitPlan(int64_t D, int64_t N, int64_t T, int smCount) {
  SplitPlan p = {};
  const int64_t tilesN = (N + kTileN - 1) / kTileN;
  p.mb = 2 * ((D + 255) / 256) * tilesN >= smCount ? 2 : 1;
  p.tilesM = static_cast<int>((D + 128 * p.mb - 1) / (128 * p.mb));
  p.tilesN = static_cast<int>(tilesN);
  p.kBlocks = static_cast<int>((T + kTokens - 1) / kTokens);
  const int64_t tiles = static_cast<int64_t>(p.tilesM) * p.tilesN;
  int64_t splits = std::max<int64_t>(1, std::min<int64_t>(smCount / std::max<int64_t>(1, tiles), p.kBlocks / 8));
  p.kPerSplit = static_cast<int>((p.kBlocks + splits - 1) / splits);
  p.splits = p.kPerSplit > 0 ? (p.kBlocks + p.kPerSplit - 1) / p.kPerSplit : 1;
  return p;
}

void gradFail(char *errorText, const char *msg) {
  if (errorText) std::snprintf(errorText, 256, "%s", msg);
}

template <int ELEM, int OUT, int MB>
int launchGradVariant(const CUtensorMap &dy, const GradParams &p, int grid, cudaStream_t stream) {
  auto kernel = checkpointGradKernel<ELEM, OUT, MB>;
  static PerDeviceOnce reserved;
  const cudaError_t e = reserved.run([&] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(gradSmemBytes<MB>()));
  });
  if (e != cudaSuccess) return e;
  return launchOrdinary(kernel, dim3(static_cast<unsigned int>(grid)), dim3(kThreads), gradSmemBytes<MB>(), stream, dy, p);
}
template <int ELEM> int launchGradTyped(int out, int mb, const CUtensorMap &dy, const GradParams &p, int grid, cudaStream_t stream) {
  if (out == kF32)
    return mb == 2 ? launchGradVariant<ELEM, kF32, 2>(dy, p, grid, stream) : launchGradVariant<ELEM, kF32, 1>(dy, p, grid, stream);
  return mb == 2 ? launchGradVariant<ELEM, ELEM, 2>(dy, p, grid, stream) : launchGradVariant<ELEM, ELEM, 1>(dy, p, grid, stream);
}

} // namespace

size_t checkpointGradWorkspaceBytes(int64_t cols, int64_t outCols, int64_t rows, int smCount) {
  const SplitPlan p = splitPlan(cols, outCols, rows, smCount);
  return p.splits > 1 ? static_cast<size_t>(p.splits) * static_cast<size_t>(cols) * static_cast<size_t>(outCols) * sizeof(float) : 0;
}

int launchCheckpointGrad(const CheckpointGradLaunch &l, cudaStream_t stream, int *launched, char *errorText) {
  if (launched) *launched = 0;
  if (l.cols == 0 || l.outCols == 0) return 0;
  const int64_t ob = l.outType == kF32 ? 4 : 2;
  if (l.elemType != kF16 && l.elemType != kBF16) { gradFail(errorText, "checkpoint gradient: dy is f16 or bf16"); return 1; }
  if (l.accumulate && l.outType != kF32) { gradFail(errorText, "checkpoint gradient: only an f32 output is added to"); return 1; }
  if (l.cols % 16 || l.outCols % 8 || l.in.codesLd % 16 || (l.dy.ld * 2) % 16 || (l.out.ld * ob) % 16) {
    gradFail(errorText, "checkpoint gradient: D a multiple of 16, N of 8, and 16-byte row lengths (TMA tensor maps)");
    return 1;
  }
  if ((reinterpret_cast<uintptr_t>(l.in.codes) | reinterpret_cast<uintptr_t>(l.dy.base) | reinterpret_cast<uintptr_t>(l.out.base)) & 15u) {
    gradFail(errorText, "checkpoint gradient: codes, dy and dweight must be 16-byte aligned");
    return 1;
  }
  if (l.statusWord < 0 || l.statusWord >= kCheckpointGradStatusWords) { gradFail(errorText, "checkpoint gradient: no such status word"); return 1; }
  if (l.rows >= (1ll << 31) - kTokens || l.cols >= (1ll << 30) || l.outCols >= (1ll << 30)) { gradFail(errorText, "checkpoint gradient: dimension too large"); return 1; }
  if (l.rows == 0) {  // a sum of nothing
    if (l.accumulate) return 0;
    return cudaMemset2DAsync(l.out.base, static_cast<size_t>(l.out.ld * ob), 0, static_cast<size_t>(l.outCols * ob), static_cast<size_t>(l.cols), stream);
  }
  int device = 0;
  if (const cudaError_t e = cudaGetDevice(&device); e != cudaSuccess) return e;
  const int sms = deviceSmCount(device);
  const SplitPlan plan = splitPlan(l.cols, l.outCols, l.rows, sms);
  if (static_cast<int64_t>(plan.tilesM) * plan.tilesN * plan.splits >= (1ll << 31)) { gradFail(errorText, "checkpoint gradient: dimension too large"); return 1; }
  const size_t need = checkpointGradWorkspaceBytes(l.cols, l.outCols, l.rows, sms);
  if (need && (!l.workspace || l.workspaceBytes < need)) { gradFail(errorText, "checkpoint gradient: workspace too small"); return 1; }

  CUtensorMap mapDy;
  const CUtensorMapDataType dt = l.elemType == kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  if (!makeMap2d(&mapDy, dt, l.dy.base, static_cast<uint64_t>(l.outCols), static_cast<uint64_t>(l.rows), static_cast<uint64_t>(l.dy.ld) * 2, 64, kTokens)) {
    gradFail(errorText, "checkpoint gradient: cuTensorMapEncodeTiled failed (driver entry point missing or bad operand layout)");
    return 1;
  }
  GradParams p = {};
  p.D = static_cast<int>(l.cols);
  p.N = static_cast<int>(l.outCols);
  p.T = static_cast<int>(l.rows);
  p.tilesM = plan.tilesM;
  p.tilesN = plan.tilesN;
  p.kBlocks = plan.kBlocks;
  p.splits = plan.splits;
  p.kPerSplit = plan.kPerSplit;
  p.band = 16;
  p.codes = l.in.codes;
  p.codesLd = l.in.codesLd;
  p.exps = l.in.exps;
  p.expsLd = l.in.expsLd;
  p.statusWord = l.statusWord;
  const bool joined = plan.splits > 1;
  p.out = joined ? l.workspace : l.out.base;
  p.outLd = joined ? l.outCols : l.out.ld;
  p.splitStride = joined ? l.cols * l.outCols : 0;
  p.accumulate = joined ? 0 : l.accumulate;
  const unsigned int fmt = l.elemType == kF16 ? 0u : 1u;
  // D f32, A and B of the same 16-bit type, both with the long side contiguous (bits 15 and 16), 128 x 256
  p.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 15) | (1u << 16) | ((kTileN >> 3) << 17) | ((128u >> 4) << 24);
  const int grid = std::min(sms, plan.tilesM * plan.tilesN * plan.splits);
  const int out = joined ? static_cast<int>(kF32) : l.outType;
  int rc = l.elemType == kF16 ? launchGradTyped<kF16>(out, plan.mb, mapDy, p, grid, stream)
                              : launchGradTyped<kBF16>(out, plan.mb, mapDy, p, grid, stream);
  if (rc != 0) return rc;
  if (launched) *launched += 1;
  if (joined) {
    const int64_t quads = l.cols * l.outCols / 4;
    const unsigned int joinGrid = static_cast<unsigned int>(std::min<int64_t>((quads + 255) / 256, static_cast<int64_t>(sms) * 16));
    const float *partial = static_cast<const float *>(l.workspace);
    const auto kernel = l.outType == kF32 ? checkpointGradJoinKernel<kF32> : l.outType == kF16 ? checkpointGradJoinKernel<kF16> : checkpointGradJoinKernel<kBF16>;
    rc = launchOrdinary(kernel, dim3(joinGrid), dim3(256), 0, stream, partial, plan.splits, l.cols, static_cast<int>(l.outCols), l.out.base, l.out.ld, l.accumulate);
    if (rc == 0 && launched) *launched += 1;
  }
  return rc;
}

int checkpointGradCheckStatus(int word, char *errorText) {
  unsigned int status = 0;
  const size_t at = static_cast<size_t>(word) * sizeof(status);
  cudaError_t e = cudaMemcpyFromSymbol(&status, checkpointGradStatusWords, sizeof(status), at);
  if (e == cudaSuccess && status == 0) return 0;
  if (e != cudaSuccess) {
    if (errorText) std::snprintf(errorText, 256, "checkpoint gradient: status read failed: %s", cudaGetErrorString(e));
    return 1;
  }
  const unsigned int zero = 0;
  cudaMemcpyToSymbol(checkpointGradStatusWords, &zero, sizeof(zero), at);
  static const char *roles[] = {"TMA producer", "MMA issuer", "output", "conversion"};
  if (errorText)
    std::snprintf(errorText, 256, "checkpoint gradient: %s gave up waiting on a pipeline barrier after 2 s (status 0x%x)", roles[std::min(3u, status & 0xffu)], status);
  return 1;
}

} // namespace kernels
} // namespace afir
