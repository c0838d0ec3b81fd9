// 16-bit products of the linear layer on pairs of SMs (tcgen05 cta_group::2).
//
// Two CTAs of a cluster share one 256 x BN tile: each holds 128 rows of A, half of B's
// BN rows and the accumulators of its 128 rows, so every operand byte in shared memory
// feeds twice the products of a single-SM tile.  TMA brings the operand tiles (zeros
// outside the operand) into a ring of stages; one thread of the leading CTA issues the
// MMAs of both; eight epilogue warps per CTA empty the accumulators, of which TMEM holds
// two sets.
//
// Bound by the tensor cores.  bf16, 16,384 x 4,096 x 4,096 (550 GFLOP a product): d W 345 us
// (1.59 PFLOP/s, 0.95 of the measured burst rate), x W^T with SiLU, residual and p 385 us, d^T x
// 390 us (256 tiles are 3.5 waves of 74 pairs).  Kernel times of short bursts; a long run of whole calls is some 15% slower.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "dense_epilogue.cuh"
#include "tcgen05.cuh"
#include "tmap.cuh"

namespace ictc {

// ------------------------------------------------------------------ pair primitives

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

// Cluster-space address of the same shared-memory object in CTA `rank`.
__device__ __forceinline__ uint32_t peer_addr(const void* p, uint32_t rank) {
  uint32_t out;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(smem_addr(p)), "r"(rank));
  return out;
}

__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar)
               : "memory");
}

__device__ __forceinline__ void pair_tmem_alloc(uint32_t* out, uint32_t columns) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                   smem_addr(out)),
               "r"(columns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void pair_tmem_free(uint32_t addr, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns)
               : "memory");
}

__device__ __forceinline__ void pair_mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t desc,
                                             bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(desc), "r"(static_cast<uint32_t>(add))
      : "memory");
}

// One arrival on `bar` of both CTAs when the MMAs issued so far have finished.
__device__ __forceinline__ void pair_commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
      " [%0], %1;" ::"r"(smem_addr(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}

// 2-D tile load into this CTA's shared memory; its bytes complete on the barrier at the
// cluster address `bar`, this CTA's or its pair's.
__device__ __forceinline__ void pair_load_2d(void* dst, const CUtensorMap* map, int x, int y,
                                             uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile"
      ".mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      ::"r"(smem_addr(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

// ------------------------------------------------------------------------ the product

constexpr int kPairRows = 256;  // rows of A per pair
constexpr int kPairEpilogueWarps = 8;
constexpr int kPairLoadWarp = kPairEpilogueWarps, kPairMmaWarp = kPairEpilogueWarps + 1;
constexpr int kPairThreads = (kPairMmaWarp + 1) * 32;

template <int BN>
constexpr int kPairStageBytes = (128 + BN / 2) * 128;

// As many stages as shared memory holds beside the epilogue's staging.
template <int BN>
constexpr int kPairStages = BN == 256 ? 6 : 8;

template <int BN>
constexpr size_t kPairSmem =
    1024 + kPairStages<BN> * kPairStageBytes<BN> + kPairEpilogueWarps * 4096 + 256;

// Box of an operand's tensor map: K-major {64 k, rows}, MN-major {64 rows, 64 k}.
struct alignas(64) OperandMaps {
  CUtensorMap a, b;
};

template <bool MN, int ROWS>
__device__ __forceinline__ void load_tile(unsigned char* dst, const CUtensorMap* map, int mn0,
                                          int k0, uint32_t bar) {
  if constexpr (MN) {
#pragma unroll
    for (int j = 0; j < ROWS / 64; ++j) pair_load_2d(dst + j * 8192, map, mn0 + j * 64, k0, bar);
  } else {
    pair_load_2d(dst, map, k0, mn0, bar);
  }
}

template <typename T, bool A_MN, bool B_MN, int BN, int ACT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    pair_product_kernel(const __grid_constant__ OperandMaps maps, const __grid_constant__ ProductArgs p) {
  constexpr int S = kPairStages<BN>;
  constexpr uint32_t kABytes = 128 * 128;
  constexpr uint32_t kColumns = 2 * BN;  // two accumulator sets
  extern __shared__ unsigned char raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t{1023});
  unsigned char* staging = smem + S * kPairStageBytes<BN>;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + kPairEpilogueWarps * 4096);  // leader's
  uint64_t* empty = full + S;
  uint64_t* done = empty + S;
  uint64_t* room = done + 2;  // leader's
  uint64_t* drain = room + 2;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(drain + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&done[s], 1);
      mbar_init(&room[s], 2 * kPairEpilogueWarps);
    }
    mbar_init(drain, 1);
    fence_mbarrier_init();
  }
  if (warp == kPairMmaWarp) pair_tmem_alloc(tmem_at, kColumns);
  tcgen05_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers are ready before either signals the other's
  tcgen05_fence_after();
  const uint32_t tmem = *tmem_at;
  const int64_t total = static_cast<int64_t>(p.tiles_m) * p.tiles_n * p.splits;
  const int64_t first = blockIdx.x >> 1, step = gridDim.x >> 1;

  if (warp == kPairLoadWarp) {
    if (lane == 0) {
      bool ok = true;
      uint32_t it = 0;
      for (int64_t t = first; ok && t < total; t += step) {
        const TilePos pos = tile_at<kPairRows>(p, t, BN);
        const int m0 = static_cast<int>(pos.m0) + rank * 128;
        const int n0 = static_cast<int>(pos.n0) + rank * (BN / 2);
        for (int c = pos.c0; c < pos.c1; ++c, ++it) {
          const int s = it % S;
          ok = mbar_wait_idle(&empty[s], ((it / S) & 1) ^ 1, kCodeProducer);
          if (!ok) break;
          unsigned char* stage = smem + s * kPairStageBytes<BN>;
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * kPairStageBytes<BN>);
          const uint32_t bar = peer_addr(&full[s], 0);
          load_tile<A_MN, 128>(stage, &maps.a, m0, c * 64, bar);
          load_tile<B_MN, BN / 2>(stage + kABytes, &maps.b, n0, c * 64, bar);
        }
      }
      // every stage's release by the MMAs has arrived before the CTA goes away
      for (int i = 0; ok && i < S; ++i, ++it)
        ok = mbar_wait_idle(&empty[it % S], ((it / S) & 1) ^ 1, kCodeProducer);
      if (!ok) {  // give copies in flight time to land before the CTA goes away
        const unsigned long long start = global_timer_ns();
        while (global_timer_ns() - start < kDrainLimitNs) {
        }
      }
    }
    __syncwarp();
  } else if (warp == kPairMmaWarp) {
    if (rank == 0 && lane == 0) {
      constexpr uint32_t kDesc =
          mma_descriptor(std::is_same_v<T, __nv_bfloat16>, A_MN, B_MN, kPairRows, BN);
      bool ok = true;
      uint32_t it = 0, set = 0;
      for (int64_t t = first; ok && t < total; t += step, ++set) {
        const TilePos pos = tile_at<kPairRows>(p, t, BN);
        ok = mbar_wait_idle(&room[set & 1], ((set >> 1) & 1) ^ 1, kCodeMma);
        if (!ok) break;
        tcgen05_fence_after();
        const uint32_t d = tmem + (set & 1) * BN;
        for (int c = pos.c0; c < pos.c1; ++c, ++it) {
          const int s = it % S;
          ok = mbar_wait_idle(&full[s], (it / S) & 1, kCodeMma);
          if (!ok) break;
          tcgen05_fence_after();
          const uint32_t sa = smem_addr(smem + s * kPairStageBytes<BN>);
          const uint64_t da = matrix_descriptor(sa, 8192, 1024);
          const uint64_t db = matrix_descriptor(sa + kABytes, 8192, 1024);
#pragma unroll
          for (int k = 0; k < 4; ++k)  // the descriptor's address field counts 16 bytes
            pair_mma_f16(d, da + k * (A_MN ? 128 : 2), db + k * (B_MN ? 128 : 2), kDesc,
                         c > pos.c0 || k > 0);
          pair_commit(&empty[s]);
        }
        if (!ok) break;
        pair_commit(&done[set & 1]);
      }
      if (!ok) {
        pair_commit(drain);
        mbar_wait(drain, 0, kCodeDrain, kDrainLimitNs);
      }
    }
    __syncwarp();
  } else {
    const int quad = warp & 3, half = warp >> 2;
    constexpr int kHalf = BN / 2;
    float4* mine = reinterpret_cast<float4*>(staging + warp * 4096);
    bool ok = true;
    uint32_t set = 0;
    for (int64_t t = first; t < total; t += step, ++set) {
      const TilePos pos = tile_at<kPairRows>(p, t, BN);
      const int64_t row0 = pos.m0 + rank * 128 + quad * 32, col0 = pos.n0 + half * kHalf;
      ResidualBlock<T> res, next;
      load_residual(p, row0, col0, lane, next);
      ok = mbar_wait_warp(&done[set & 1], (set >> 1) & 1, kCodeEpilogue);
      if (!ok) break;
      tcgen05_fence_after();
      const uint32_t at =
          tmem + (set & 1) * BN + (static_cast<uint32_t>(quad * 32) << 16) + half * kHalf;
#pragma unroll 1
      for (int cb = 0; cb < kHalf / 32; ++cb) {
        float acc[32];
        float(&lo)[16] = *reinterpret_cast<float(*)[16]>(acc);
        float(&hi)[16] = *reinterpret_cast<float(*)[16]>(acc + 16);
        tmem_load16(at + cb * 32, lo);
        tmem_load16(at + cb * 32 + 16, hi);
        res = next;
        const bool last = cb == kHalf / 32 - 1;
        if (!last) load_residual(p, row0, col0 + (cb + 1) * 32, lane, next);
        tmem_load_wait();
        if (last) {  // the set's last columns are in registers
          tcgen05_fence_before();
          __syncwarp();
          if (lane == 0) arrive_cluster(peer_addr(&room[set & 1], 0));
        }
        write_block<T, ACT>(p, pos.split, acc, mine, row0, col0 + cb * 32, lane, res);
      }
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  cluster_sync();  // neither CTA leaves while the other may still signal it
  if (warp == kPairMmaWarp) {
    tcgen05_fence_after();
    pair_tmem_free(tmem, kColumns);
  }
}

}  // namespace ictc
