// Float32 products of the linear layer with operands that TMA can address.
//
// C = A B^T by six products of bf16 parts (dense_linear.cu).  Four kinds of warps: one
// thread brings raw operand tiles, 32 elements of K at a time, by TMA (zeros outside the
// operand) into a ring of slots; eight producer warps cut them into parts in the swizzled
// order that the MMA reads; one thread issues the MMAs; eight epilogue warps move sums out
// of TMEM, which holds two sets, every 256 elements of K.
//
// What bounds it: no single unit (65,536 x 128 x 512: the tensor pipe is busy 19% to 34% of
// the time, LSU wavefronts 40% to 48%, issue slots 37% to 54%, DRAM 20% to 28%), so the chain
// raw tile, cut, MMA, accumulator.  An MMA fetches its operands from shared memory every time:
// six of a 128 x 128 tile's step of 16 read 6 x 8 KB; meeting b1 | b2 in one MMA with a1 saves
// one reading of A.  A 64-column tile meets b1 | b2 | b3 at once and needs three MMAs.
//  65,536 x 128 x 512: forward with gelu and p 118
// us (73 TFLOP/s of float32 products), d W 84 us, d^T x 67 us (128 TFLOP/s); with operands
// staged through registers 182, 109 and 95.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "dense_epilogue.cuh"
#include "dense_pair.cuh"
#include "tcgen05.cuh"
#include "tmap.cuh"

namespace ictc {

// Warpgroups: two of epilogue warps, two of producers, one with the MMA and the load
// warp.  Registers move from the others to the epilogue, which holds a tile's sums.
constexpr int kCutEpilogueWarps = 8, kCutProducerWarps = 8;
constexpr int kCutMmaWarp = 16, kCutLoadWarp = 17;
constexpr int kCutThreads = 20 * 32;
constexpr int kCutLaunchRegisters = 96;  // 65,536 / 640, in steps of 8
constexpr int kCutEpilogueRegisters = 152, kCutProducerRegisters = 64, kCutIssueRegisters = 48;
static_assert(kCutEpilogueWarps * kCutEpilogueRegisters +
                  kCutProducerWarps * kCutProducerRegisters + 4 * kCutIssueRegisters <=
              20 * kCutLaunchRegisters);

template <int N>
__device__ __forceinline__ void take_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void give_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
constexpr int kCutK = 32;           // K elements of a raw slot and of a half of the cut tile
constexpr int kCutGroupHalves = 8;  // halves (256 elements of K) between moves out of TMEM

template <int BN>
constexpr uint32_t kCutRaw = (128 + BN) * kCutK * 4;
template <int BN>
constexpr int kCutSlots = BN == 128 ? 3 : 4;
template <int BN>
constexpr uint32_t kCutTile = 3 * (128 + BN) * 128;
template <int BN>
constexpr size_t kCutSmem =
    1024 + kCutTile<BN> + kCutSlots<BN> * kCutRaw<BN> + kCutEpilogueWarps * 4096 + 256;

// Cuts one raw operand tile into half `h` of its place in the cut tile ([3 parts][ROWS x
// 128 bytes]).  A lane takes four consecutive elements.  K-major: raw rows are 32 elements
// (128 bytes); two of a warp's four rows have bit 2 of their index set, so that the half
// rows they write fall on all banks.  MN-major: raw rows are ROWS elements of one k.
template <bool MN, int ROWS>
__device__ __forceinline__ void cut_tile(const unsigned char* raw, unsigned char* dst, int h,
                                         int tid) {
  constexpr int kThreads = kCutProducerWarps * 32;
  constexpr int kUnits = ROWS * kCutK / 4 / kThreads;  // per thread
  const int warp = tid >> 5, lane = tid & 31;
  float4 f[kUnits];
  uint32_t to[kUnits];
  // all loads ahead of the stores, which might alias them
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    uint32_t from;
    if constexpr (MN) {
      constexpr int kPerK = ROWS / 4;  // units of a k: 32 or 16
      const int at = i * kThreads + tid, k = at / kPerK, u = at % kPerK;
      from = (k * ROWS + 4 * u) * 4;
      to[i] = (u >> 4) * 8192 + swizzled(h * kCutK + k, (u & 15) >> 1) + (u & 1) * 8;
    } else {
      const int j = lane >> 3, u = lane & 7, w = warp + i * kCutProducerWarps;  // four rows each
      const int r = (w >> 2) * 16 + ((w >> 1) & 1) * 8 + (j & 1) * 4 + (w & 1) * 2 + (j >> 1);
      from = (r * kCutK + 4 * u) * 4;
      to[i] = swizzled(r, h * 4 + (u >> 1)) + (u & 1) * 8;
    }
    f[i] = *reinterpret_cast<const float4*>(raw + from);
  }
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    uint32_t lo[3], hi[3];
    cut_pair(f[i].x, f[i].y, lo);
    cut_pair(f[i].z, f[i].w, hi);
#pragma unroll
    for (int q = 0; q < 3; ++q)
      *reinterpret_cast<uint2*>(dst + q * ROWS * 128 + to[i]) = make_uint2(lo[q], hi[q]);
  }
}

template <bool MN, int ROWS>
__device__ __forceinline__ void load_raw(unsigned char* dst, const CUtensorMap* map, int64_t mn0,
                                         int k0, uint64_t* bar) {
  if constexpr (MN) tma_load_2d(dst, map, static_cast<int>(mn0), k0, bar);
  else tma_load_2d(dst, map, k0, static_cast<int>(mn0), bar);
}

template <bool A_MN, bool B_MN, int BN, int ACT>
__global__ void __launch_bounds__(kCutThreads, 1)
    cut_product_kernel(const __grid_constant__ OperandMaps maps,
                       const __grid_constant__ ProductArgs p) {
  constexpr int R = kCutSlots<BN>;
  constexpr uint32_t kA = 3 * 128 * 128;  // bytes of A's parts
  constexpr uint32_t kSet = BN == 128 ? 256 : 192;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* tile = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t{1023});
  unsigned char* slots = tile + kCutTile<BN>;
  unsigned char* staging = slots + R * kCutRaw<BN>;
  uint64_t* raw_full = reinterpret_cast<uint64_t*>(staging + kCutEpilogueWarps * 4096);
  uint64_t* raw_empty = raw_full + R;
  uint64_t* full = raw_empty + R;  // halves of the cut tile
  uint64_t* empty = full + 2;
  uint64_t* done = empty + 2;
  uint64_t* room = done + 2;
  uint64_t* drain = room + 2;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(drain + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < R; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], kCutProducerWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&full[i], kCutProducerWarps);
      mbar_init(&empty[i], 1);
      mbar_init(&done[i], 1);
      mbar_init(&room[i], kCutEpilogueWarps);
    }
    mbar_init(drain, 1);
    fence_mbarrier_init();
  }
  if (warp == 0) tmem_alloc(tmem_at, 512);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = *tmem_at;
  const int64_t total = static_cast<int64_t>(p.tiles_m) * p.tiles_n * p.splits;
  // halves [h0, h1) of 32 elements of K of a work item
  const auto halves_end = [&](const TilePos& pos) {
    const int64_t all = (p.k + kCutK - 1) / kCutK;
    return 2ll * pos.c1 < all ? 2ll * pos.c1 : all;
  };

  if (warp >= kCutMmaWarp) {
    give_registers<kCutIssueRegisters>();
    if (warp == kCutLoadWarp && lane == 0) {
      bool ok = true;
      uint32_t n = 0;
      for (int64_t t = blockIdx.x; ok && t < total; t += gridDim.x) {
        const TilePos pos = tile_at<128>(p, t, BN);
        const int64_t h1 = halves_end(pos);
        for (int64_t h = 2ll * pos.c0; h < h1; ++h, ++n) {
          const int s = n % R;
          ok = mbar_wait_idle(&raw_empty[s], ((n / R) & 1) ^ 1, kCodeProducer);
          if (!ok) break;
          unsigned char* slot = slots + s * kCutRaw<BN>;
          mbar_arrive_expect_tx(&raw_full[s], kCutRaw<BN>);
          load_raw<A_MN, 128>(slot, &maps.a, pos.m0, static_cast<int>(h * kCutK), &raw_full[s]);
          load_raw<B_MN, BN>(slot + 128 * kCutK * 4, &maps.b, pos.n0,
                             static_cast<int>(h * kCutK), &raw_full[s]);
        }
      }
      if (!ok) {  // copies in flight land before the CTA goes away
        const unsigned long long begin = global_timer_ns();
        while (global_timer_ns() - begin < kDrainLimitNs) {
        }
      }
    }
    if (warp == kCutMmaWarp && lane == 0) {
      constexpr uint32_t kOne = mma_descriptor(true, A_MN, B_MN, 128, BN);
      constexpr uint32_t kTwo = mma_descriptor(true, A_MN, B_MN, 128, 2 * BN);
      constexpr uint32_t kThree = mma_descriptor(true, A_MN, B_MN, 128, BN == 64 ? 192 : 128);
      // strides in the descriptors' 16-byte units: a step of 16 elements, a part
      constexpr uint64_t kAs = A_MN ? 128 : 2, kBs = B_MN ? 128 : 2;
      constexpr uint64_t kAp = 128 * 8, kBp = BN * 8;
      const uint64_t a0 = matrix_descriptor(smem_addr(tile), 8192, 1024);
      const uint64_t b0 = matrix_descriptor(smem_addr(tile + kA), 8192, 1024);
      bool ok = true;
      uint32_t n = 0, set = 0;
      for (int64_t t = blockIdx.x; ok && t < total; t += gridDim.x) {
        const TilePos pos = tile_at<128>(p, t, BN);
        const int64_t h0 = 2ll * pos.c0, h1 = halves_end(pos);
        for (int64_t h = h0; h < h1; ++h, ++n) {
          const bool first = (h - h0) % kCutGroupHalves == 0;
          if (first) ok = mbar_wait_idle(&room[set & 1], ((set >> 1) & 1) ^ 1, kCodeMma);
          if (ok) ok = mbar_wait_idle(&full[n & 1], (n >> 1) & 1, kCodeMma);
          if (!ok) break;
          tcgen05_fence_after();
          const uint32_t d = tmem + (set & 1) * kSet;
          const int64_t left = p.k - h * kCutK;
          const int steps = left > 16 ? 2 : 1;
          bool add = !first;
          for (int q = 0; q < steps; ++q) {
            const uint64_t a = a0 + (2 * (n & 1) + q) * kAs, b = b0 + (2 * (n & 1) + q) * kBs;
            if constexpr (BN == 128) {
              mma_f16(d, a, b, kTwo, add);  // a1 (b1 | b2): large and small sums side by side
              mma_f16(d + BN, a + 2 * kAp, b, kOne, true);
              mma_f16(d + BN, a, b + 2 * kBp, kOne, true);
              mma_f16(d + BN, a + kAp, b + kBp, kOne, true);
              mma_f16(d + BN, a + kAp, b, kOne, true);
            } else {
              mma_f16(d, a, b, kThree, add);
              mma_f16(d + BN, a + kAp, b, kTwo, true);
              mma_f16(d + 2 * BN, a + 2 * kAp, b, kOne, true);
            }
            add = true;
          }
          mma_commit(&empty[n & 1]);
          if (h + 1 == h1 || (h + 1 - h0) % kCutGroupHalves == 0) {
            mma_commit(&done[set & 1]);
            ++set;
          }
        }
      }
      if (!ok) {  // MMAs in flight finish
        mma_commit(drain);
        mbar_wait(drain, 0, kCodeDrain, kDrainLimitNs);
      }
    }
    __syncwarp();
  } else if (warp >= kCutEpilogueWarps) {
    give_registers<kCutProducerRegisters>();
    const int tid = threadIdx.x - kCutEpilogueWarps * 32;
    bool ok = true;
    uint32_t n = 0;
    for (int64_t t = blockIdx.x; ok && t < total; t += gridDim.x) {
      const TilePos pos = tile_at<128>(p, t, BN);
      const int64_t h1 = halves_end(pos);
      for (int64_t h = 2ll * pos.c0; h < h1; ++h, ++n) {
        const int s = n % R, half = n & 1;
        ok = mbar_wait_warp(&raw_full[s], (n / R) & 1, kCodeProducer) &&
             mbar_wait_warp(&empty[half], ((n >> 1) & 1) ^ 1, kCodeProducer);
        if (!ok) break;
        const unsigned char* slot = slots + s * kCutRaw<BN>;
        cut_tile<A_MN, 128>(slot, tile, half, tid);
        cut_tile<B_MN, BN>(slot + 128 * kCutK * 4, tile + kA, half, tid);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&raw_empty[s]);
          mbar_arrive(&full[half]);
        }
      }
    }
  } else {
    take_registers<kCutEpilogueRegisters>();
    constexpr int kHalf = BN / 2;
    const int quad = warp & 3, half = warp >> 2;
    float4* mine = reinterpret_cast<float4*>(staging + warp * 4096);
    bool ok = true;
    uint32_t set = 0;
    for (int64_t t = blockIdx.x; ok && t < total; t += gridDim.x) {
      const TilePos pos = tile_at<128>(p, t, BN);
      const int64_t h0 = 2ll * pos.c0, h1 = halves_end(pos);
      const int groups = static_cast<int>((h1 - h0 + kCutGroupHalves - 1) / kCutGroupHalves);
      const int64_t row0 = pos.m0 + quad * 32;
      ResidualBlock<float> res;  // early where registers allow
      if constexpr (BN == 64) load_residual(p, row0, pos.n0 + half * kHalf, lane, res);
      float acc[kHalf];
      for (int gi = 0; gi < groups; ++gi, ++set) {
        ok = mbar_wait_warp(&done[set & 1], (set >> 1) & 1, kCodeEpilogue);
        if (!ok) break;
        tcgen05_fence_after();
        const uint32_t at =
            tmem + (set & 1) * kSet + (static_cast<uint32_t>(quad * 32) << 16) + half * kHalf;
#pragma unroll
        for (int j = 0; j < kHalf; j += 16) {
          float w[16], y[16];
          tmem_load16(at + BN + j, y);
          if constexpr (BN == 64) {
            tmem_load16(at + 2 * BN + j, w);
            tmem_load_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] += w[i];
          }
          tmem_load16(at + j, w);
          tmem_load_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = join_parts(w[i], y[i]);
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[j + i] = gi == 0 ? w[i] : acc[j + i] + w[i];
        }
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&room[set & 1]);
      }
      if (!ok) break;
#pragma unroll
      for (int cb = 0; cb < kHalf / 32; ++cb) {
        const int64_t col0 = pos.n0 + half * kHalf + cb * 32;
        stage_block(acc + cb * 32, mine, lane);
        write_staged<float, ACT, BN == 128>(p, pos.split, mine, row0, col0, lane, res);
      }
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 0) {
    tcgen05_fence_after();
    tmem_free(tmem, 512);
  }
}

}  // namespace ictc
