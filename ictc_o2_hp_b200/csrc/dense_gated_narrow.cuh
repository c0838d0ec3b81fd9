// Gated linear layers of at most 64 inputs and 64 outputs over many rows (radial networks over
// edges): forward and the whole backward as one kernel each.
//
// Bound by HBM and the issue slots, so nothing but x, g, y and dx moves: the forward keeps no
// p, and the backward computes it again from x, whose tile it needs in shared memory for dW
// anyway.  (Kept in float32, p would be two thirds of the training step's traffic.)  W is cut
// and laid out in shared memory once per CTA, gate rows 0-63 and up rows 64-127, and serves p
// = x W^T as a K-major and dx = D W as an MN-major operand; D, formed from p in TMEM by threads
// that own a row each, serves D W as a K-major and D^T x as an MN-major operand.
//
//   p  = x W^T   M = 128 rows, N = 128 (gate | up), reduction over k <= 64
//   dx = D W     M = 128 rows, N = 64, reduction over the 128 columns of D
//   dW = D^T x   M = 128 columns of D, N = 64, reduction over the tile's 128 rows
//
// A float32 product has two sums in TMEM, of a1 b1 and of the five other partial products;
// both of dx, dW (two tiles of it, because the tensor core truncates when it adds) and p take
// all 512 columns.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "dense_cut.cuh"
#include "dense_epilogue.cuh"
#include "dense_narrow.cuh"
#include "tcgen05.cuh"

namespace ictc {

constexpr int kGatedRows = 2 * kNarrow;          // of W, and columns of D
constexpr uint32_t kGatedBlock = kNarrowTile * 128;  // 64 columns of 128 rows, one part

template <typename T>
constexpr uint32_t kGatedOperand = kCut<T> * kGatedBlock;

struct GatedNarrowArgs {
  const void *x, *w, *g, *bias;  // x [m, k], w [2 n, k] (rows ldw apart), g [m, n], bias [2 n] or null
  int64_t m, ldw;
  int n, k, tiles;
  float* partial;  // backward: [gridDim.x][2 n k + 2 n]: dW, db, or null
  Epilogue e;      // forward: y; backward: dx, or null
};

// Whole warp: eight consecutive columns of the warp's 32 TMEM lanes.
__device__ __forceinline__ void tmem_load8(uint32_t addr, float (&v)[8]) {
  uint32_t u[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]),
                 "=r"(u[6]), "=r"(u[7])
               : "r"(addr)
               : "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(u[i]);
}

// W as [128][64 k], zeros outside; THREADS threads.
template <typename T, int THREADS>
__device__ __forceinline__ void load_gated_weights(unsigned char* dst, const GatedNarrowArgs& p) {
  const T* w = static_cast<const T*>(p.w);
  for (int i = threadIdx.x; i < kGatedRows * 16; i += THREADS) {
    const int r = i >> 4, u = i & 15, c = r & (kNarrow - 1);
    const T* row = w + ((r >= kNarrow ? p.n : 0) + c) * p.ldw;
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      v[j] = c < p.n && 4 * u + j < p.k ? to_float(row[4 * u + j]) : 0.f;
    store_unit<T>(dst, kGatedRows * 128, r, u, v);
  }
}

// One K step of 16: N columns of leading sums at d, and with three parts N of the others
// behind them.  Strides of parts in the descriptors' units of 16 bytes.
template <int P, int N>
__device__ __forceinline__ void issue_gated(uint32_t d, uint64_t a, uint64_t a_part, uint64_t b,
                                            uint64_t b_part, bool bf16, bool a_mn, bool b_mn,
                                            bool add) {
  const uint32_t one = mma_descriptor(bf16, a_mn, b_mn, kNarrowTile, N);
  if constexpr (P == 3) {
    mma_f16(d, a, b, mma_descriptor(bf16, a_mn, b_mn, kNarrowTile, 2 * N), add);  // a1 (b1 | b2)
    mma_f16(d + N, a + 2 * a_part, b, one, true);
    mma_f16(d + N, a, b + 2 * b_part, one, true);
    mma_f16(d + N, a + a_part, b + b_part, one, true);
    mma_f16(d + N, a + a_part, b, one, true);
  } else {
    mma_f16(d, a, b, one, add);
  }
}

// p of a tile: K steps over k.
template <typename T>
__device__ __forceinline__ void issue_p(uint32_t d, uint32_t x_tile, uint32_t weights, int k) {
  const uint64_t a = matrix_descriptor(x_tile, 0, 1024), b = matrix_descriptor(weights, 0, 1024);
  for (int s = 0; 16 * s < k; ++s)
    issue_gated<kCut<T>, kGatedRows>(d, a + 2 * s, kGatedBlock / 16, b + 2 * s, kGatedRows * 8,
                                     !std::is_same_v<T, __half>, false, false, s > 0);
}

// Eight columns of p, of the gate's half and of the other.
template <int P>
__device__ __forceinline__ void take_p(uint32_t at, float (&gate)[8], float (&up)[8]) {
  if constexpr (P == 3) {
    float y[8], z[8];
    tmem_load8(at, gate);
    tmem_load8(at + kNarrow, up);
    tmem_load8(at + kGatedRows, y);
    tmem_load8(at + kGatedRows + kNarrow, z);
    tmem_load_wait();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      gate[i] = join_parts(gate[i], y[i]);
      up[i] = join_parts(up[i], z[i]);
    }
  } else {
    tmem_load8(at, gate);
    tmem_load8(at + kNarrow, up);
    tmem_load_wait();
  }
}

// 16 columns of a 64-column product.
template <int P>
__device__ __forceinline__ void take_product(uint32_t at, float (&v)[16]) {
  tmem_load16(at, v);
  if constexpr (P == 3) {
    float y[16];
    tmem_load16(at + kNarrow, y);
    tmem_load_wait();
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = join_parts(v[i], y[i]);
  } else {
    tmem_load_wait();
  }
}

// N columns of a row, of which `left` exist.  A thread owns a row, so lanes write rows apart:
// 16 bytes each, whose sectors L2 puts together.  (Through shared memory, with lanes along
// the columns, forward and backward took the same time and 32 KB that the slices need.)
template <typename T, int N>
__device__ __forceinline__ void store_columns(T* to, const float (&v)[N], int left, bool vec) {
  constexpr int V = 16 / sizeof(T);
  if (vec) {
#pragma unroll
    for (int i = 0; i < N; i += V) {
      Pack<T, V> o;
#pragma unroll
      for (int j = 0; j < V; ++j) o.v[j] = from_float<T>(v[i + j]);
      if (i < left) *reinterpret_cast<Pack<T, V>*>(to + i) = o;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < left) to[i] = from_float<T>(v[i]);
  }
}

// The producers' four warps: the tile's x from the ring of slices, cut, into `tile`.
template <typename T, int R>
__device__ __forceinline__ bool fill_x_tile(unsigned char* tile, const unsigned char* slices,
                                            uint64_t* raw_full, uint64_t* raw_empty, int t,
                                            const GatedNarrowArgs& p, int tid, int lane,
                                            uint32_t& n) {
  const int unit = tid & 15, r0 = tid >> 4;
  const int columns = (p.k + 15) & ~15;  // that the MMAs read
  SliceWalk at{t, 0, p.tiles, static_cast<int>(gridDim.x), p.m};
#pragma unroll 1
  for (int q = 0; q < kNarrowTile / kSliceRows; ++q, ++at.slice) {
    Slice<T> slice{nullptr, nullptr, p.k, 0, 0};
    const bool some = at.row() < p.m;
    const int slot = n % R;
    if (some) {
      if (!mbar_wait_warp(&raw_full[slot], (n / R) & 1, kCodeProducer)) return false;
      slice.raw = reinterpret_cast<const T*>(slices + slot * kSliceX<T>);
      slice.rows = at.rows();
    }
    float v[4][4];
    uint32_t seen = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      read_unit<true>(slice, r0 + 8 * j, unit, v[j]);
      seen |= unit_bits<true>(v[j]);
    }
    if (4 * unit < columns)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        store_unit<T>(tile, kGatedBlock, q * kSliceRows + r0 + 8 * j, unit, v[j]);
    if (some) {
      release_slot(&raw_empty[slot], seen, lane);
      ++n;
    }
  }
  return true;
}

// One thread: x's slices into the ring.
template <typename T, int R>
__device__ __forceinline__ void copy_slices(unsigned char* slices, uint64_t* raw_full,
                                            uint64_t* raw_empty, const GatedNarrowArgs& p) {
  const T* x = static_cast<const T*>(p.x);
  SliceWalk at{static_cast<int>(blockIdx.x), 0, p.tiles, static_cast<int>(gridDim.x), p.m};
  bool ok = true;
  for (uint32_t n = 0; !at.done(); at.next(), ++n) {
    const int slot = n % R;
    ok = mbar_wait_idle(&raw_empty[slot], ((n / R) & 1) ^ 1, kCodeProducer);
    if (!ok) break;
    const uint32_t bytes = slice_bytes<T>(p.k, at.rows());
    mbar_arrive_expect_tx(&raw_full[slot], bytes);
    bulk_g2s(slices + slot * kSliceX<T>, x + at.row() * p.k, bytes, &raw_full[slot]);
  }
  if (!ok) settle_copies();
}

// Warps of both kernels: 16 that take rows out of TMEM, four producers, MMA and copy warp.
// More of the first hide the latencies of TMEM and of the exponentials (with eight, bf16
// 1,048,576 x 64 x 64 forward 127 us, backward 482).
constexpr int kRowWarps = 16, kGatedProducerWarps = 4;
constexpr int kGatedMmaWarp = kRowWarps + kGatedProducerWarps, kGatedCopyWarp = kGatedMmaWarp + 1;
constexpr int kGatedThreads = 24 * 32;

// ------------------------------------------------------------------------- forward

constexpr int kGatedForwardSlices = 8;
template <typename T>
constexpr size_t kGatedForwardSmem =
    1024 + 3 * kGatedOperand<T> + kGatedForwardSlices * kSliceX<T> + kGatedRows * 4 + 256;

template <typename T>
__device__ __forceinline__ void stage_bias(float* to, const GatedNarrowArgs& p) {
  for (int i = threadIdx.x; i < kGatedRows; i += kGatedThreads) {
    const int c = i & (kNarrow - 1);
    to[i] = p.bias && c < p.n
                ? to_float(static_cast<const T*>(p.bias)[(i >= kNarrow ? p.n : 0) + c])
                : 0.f;
  }
}

// Eight values of the staged bias.
__device__ __forceinline__ void add_bias(float (&v)[8], const float* bias) {
  const float4 a = *reinterpret_cast<const float4*>(bias);
  const float4 b = *reinterpret_cast<const float4*>(bias + 4);
  v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
  v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
}

template <typename T, int ACT>
__global__ void __launch_bounds__(kGatedThreads, 1)
    gated_narrow_forward_kernel(const __grid_constant__ GatedNarrowArgs p) {
  constexpr int P = kCut<T>, R = kGatedForwardSlices;
  constexpr uint32_t kSet = (P == 3 ? 2 : 1) * kGatedRows;
  extern __shared__ unsigned char raw_smem[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t{1023});
  unsigned char* weights = smem;
  unsigned char* tiles = weights + kGatedOperand<T>;
  unsigned char* slices = tiles + 2 * kGatedOperand<T>;
  float* bias = reinterpret_cast<float*>(slices + R * kSliceX<T>);
  uint64_t* raw_full = reinterpret_cast<uint64_t*>(bias + kGatedRows);
  uint64_t* raw_empty = raw_full + R;
  uint64_t* full = raw_empty + R;
  uint64_t* empty = full + 2;
  uint64_t* done = empty + 2;
  uint64_t* room = done + 2;
  uint64_t* drain = room + 2;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(drain + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < R; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], kGatedProducerWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&full[i], kGatedProducerWarps);
      mbar_init(&empty[i], 1);
      mbar_init(&done[i], 1);
      mbar_init(&room[i], kRowWarps / 2);
    }
    mbar_init(drain, 1);
    fence_mbarrier_init();
  }
  if (warp == 0) tmem_alloc(tmem_at, 2 * kSet);
  load_gated_weights<T, kGatedThreads>(weights, p);
  stage_bias<T>(bias, p);
  fence_proxy_async();
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = *tmem_at;

  if (warp == kGatedCopyWarp) {
    if (lane == 0) copy_slices<T, R>(slices, raw_full, raw_empty, p);
    __syncwarp();
  } else if (warp == kGatedMmaWarp) {
    if (lane == 0) {
      bool ok = true;
      uint32_t it = 0;
      for (int t = blockIdx.x; t < p.tiles; t += gridDim.x, ++it) {
        const int s = it & 1;
        ok = mbar_wait_idle(&room[s], ((it >> 1) & 1) ^ 1, kCodeMma) &&
             mbar_wait_idle(&full[s], (it >> 1) & 1, kCodeMma);
        if (!ok) break;
        tcgen05_fence_after();
        issue_p<T>(tmem + s * kSet, smem_addr(tiles + s * kGatedOperand<T>), smem_addr(weights),
                   p.k);
        mma_commit(&empty[s]);
        mma_commit(&done[s]);
      }
      if (!ok) {  // MMAs in flight finish
        mma_commit(drain);
        mbar_wait(drain, 0, kCodeDrain, kDrainLimitNs);
      }
    }
    __syncwarp();
  } else if (warp >= kRowWarps && warp < kGatedMmaWarp) {
    const int tid = threadIdx.x - kRowWarps * 32;
    uint32_t it = 0, n = 0;  // tiles and slices so far
    for (int t = blockIdx.x; t < p.tiles; t += gridDim.x, ++it) {
      const int s = it & 1;
      if (!mbar_wait_warp(&empty[s], ((it >> 1) & 1) ^ 1, kCodeProducer) ||
          !fill_x_tile<T, R>(tiles + s * kGatedOperand<T>, slices, raw_full, raw_empty, t, p, tid,
                             lane, n))
        break;
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[s]);
    }
  } else if (warp < kRowWarps) {
    // eight warps for each of the two sets, every other tile: rows of a quad, half the columns
    const int quad = warp & 3, half = (warp >> 2) & 1, s = warp >> 3;
    T* y = static_cast<T*>(p.e.out);
    uint32_t it = 0;
    for (int t = blockIdx.x + s * gridDim.x; t < p.tiles; t += 2 * gridDim.x, ++it) {
      const int64_t row = static_cast<int64_t>(t) * kNarrowTile + quad * 32 + lane;
      if (!mbar_wait_warp(&done[s], it & 1, kCodeEpilogue)) break;
      tcgen05_fence_after();
      const uint32_t at = tmem + s * kSet + (static_cast<uint32_t>(quad * 32) << 16) + half * 32;
#pragma unroll
      for (int j = 0; j < 32; j += 8) {
        const int col = half * 32 + j;
        float gate[8], up[8];
        take_p<P>(at + j, gate, up);
        if (j == 24) {
          tcgen05_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&room[s]);
        }
        add_bias(gate, bias + col);
        add_bias(up, bias + kNarrow + col);
#pragma unroll
        for (int i = 0; i < 8; ++i) up[i] *= activate<ACT>(gate[i]);
        if (row < p.m && col < p.n) store_columns(y + row * p.n + col, up, p.n - col, p.e.vec);
      }
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 0) {
    tcgen05_fence_after();
    tmem_free(tmem, 2 * kSet);
  }
}

// ------------------------------------------------------------------------ backward

// Registers move to the row warps, which hold the sums of db.
constexpr int kGatedLaunchRegisters = 80;  // 65,536 / 768, in steps of 8
constexpr int kRowRegisters = 96, kGatedProducerRegisters = 56, kGatedIssueRegisters = 40;
static_assert(kRowWarps * kRowRegisters + kGatedProducerWarps * kGatedProducerRegisters +
                  4 * kGatedIssueRegisters <=
              24 * kGatedLaunchRegisters);
constexpr int kGatedBackwardSlices = 4;  // a tile

template <typename T>
constexpr size_t kGatedBackwardSmem = 1024 + 4 * kGatedOperand<T> +
                                      kGatedBackwardSlices * kSliceX<T> + kGatedRows * 4 + 512;

// Eight columns of D to their tile, part by part.
template <typename T>
__device__ __forceinline__ void store_d(unsigned char* at, const float (&v)[8]) {
  if constexpr (kCut<T> == 3) {
    uint32_t part[4][3];
#pragma unroll
    for (int j = 0; j < 4; ++j) cut_pair(v[2 * j], v[2 * j + 1], part[j]);
#pragma unroll
    for (int q = 0; q < 3; ++q)
      *reinterpret_cast<uint4*>(at + q * 2 * kGatedBlock) =
          make_uint4(part[0][q], part[1][q], part[2][q], part[3][q]);
  } else {
    Pack<T, 8> o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o.v[j] = from_float<T>(v[j]);
    *reinterpret_cast<Pack<T, 8>*>(at) = o;
  }
}

template <typename T, int ACT>
__global__ void __launch_bounds__(kGatedThreads, 1)
    gated_narrow_backward_kernel(const __grid_constant__ GatedNarrowArgs p) {
  constexpr int P = kCut<T>, R = kGatedBackwardSlices;
  constexpr uint32_t kOrders = P == 3 ? 2 : 1;
  constexpr uint32_t kDx = kOrders * kGatedRows, kDw = kDx + kOrders * kNarrow;
  constexpr uint32_t kColumns = kOrders * 256;
  extern __shared__ unsigned char raw_smem[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t{1023});
  unsigned char* weights = smem;
  unsigned char* x_tile = weights + kGatedOperand<T>;
  unsigned char* d_tile = x_tile + kGatedOperand<T>;  // [parts][gate, up][128 rows][64]
  unsigned char* slices = d_tile + 2 * kGatedOperand<T>;
  float* bias = reinterpret_cast<float*>(slices + R * kSliceX<T>);
  uint64_t* raw_full = reinterpret_cast<uint64_t*>(bias + kGatedRows);
  uint64_t* raw_empty = raw_full + R;
  uint64_t* x_full = raw_empty + R;
  uint64_t* x_empty = x_full + 1;
  uint64_t* p_done = x_empty + 1;
  uint64_t* p_room = p_done + 1;
  uint64_t* d_full = p_room + 1;
  uint64_t* d_empty = d_full + 1;
  uint64_t* dx_done = d_empty + 1;
  uint64_t* dx_room = dx_done + 1;
  uint64_t* dw_done = dx_room + 1;
  uint64_t* dw_room = dw_done + 1;
  uint64_t* drain = dw_room + 1;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(drain + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < R; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], kGatedProducerWarps);
    }
    mbar_init(x_full, kGatedProducerWarps);
    mbar_init(x_empty, 1);
    mbar_init(p_done, 1);
    mbar_init(p_room, kRowWarps);
    mbar_init(d_full, kRowWarps);
    mbar_init(d_empty, 1);
    mbar_init(dx_done, 1);
    mbar_init(dx_room, kRowWarps);
    mbar_init(dw_done, 1);
    mbar_init(dw_room, kRowWarps);
    mbar_init(drain, 1);
    fence_mbarrier_init();
  }
  if (warp == 0) tmem_alloc(tmem_at, kColumns);
  load_gated_weights<T, kGatedThreads>(weights, p);
  stage_bias<T>(bias, p);
  // columns of x past k and of D past n are never written, but the MMAs read them
  for (uint32_t i = threadIdx.x; i < 3 * kGatedOperand<T> / 16; i += kGatedThreads)
    reinterpret_cast<uint4*>(x_tile)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async();
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = *tmem_at;
  const bool want_dx = p.e.out != nullptr, want_dw = p.partial != nullptr;
  const auto closes_group = [&](int t, uint32_t it) {
    return it % kDwTiles == kDwTiles - 1 || t + static_cast<int>(gridDim.x) >= p.tiles;
  };
  const int wide = 2 * p.n;
  float* partial = want_dw ? p.partial + static_cast<int64_t>(blockIdx.x) * (wide * p.k + wide)
                           : nullptr;

  if (warp >= kGatedMmaWarp) {
    give_registers<kGatedIssueRegisters>();
    if (warp == kGatedCopyWarp && lane == 0) copy_slices<T, R>(slices, raw_full, raw_empty, p);
    if (warp == kGatedMmaWarp && lane == 0) {
      constexpr bool kBf16 = !std::is_same_v<T, __half>;
      const uint32_t xa = smem_addr(x_tile), da = smem_addr(d_tile), wa = smem_addr(weights);
      const uint64_t d_rows = matrix_descriptor(da, 0, 1024);            // K-major
      const uint64_t d_columns = matrix_descriptor(da, kGatedBlock, 1024);  // MN-major, two blocks
      // MN-major with the parts behind one another as further columns
      const uint64_t x_columns = matrix_descriptor(xa, kGatedBlock, 1024);
      const uint64_t w_columns = matrix_descriptor(wa, kGatedRows * 128, 1024);
      constexpr uint64_t kXp = kGatedBlock / 16, kDp = 2 * kXp, kWp = kGatedRows * 8;
      bool ok = true;
      uint32_t it = 0;
      for (int t = blockIdx.x; t < p.tiles; t += gridDim.x, ++it) {
        ok = mbar_wait_idle(x_full, it & 1, kCodeMma) &&
             mbar_wait_idle(p_room, (it & 1) ^ 1, kCodeMma);
        if (!ok) break;
        tcgen05_fence_after();
        issue_p<T>(tmem, xa, wa, p.k);
        mma_commit(p_done);
        ok = mbar_wait_idle(d_full, it & 1, kCodeMma);
        if (!ok) break;
        tcgen05_fence_after();
        // dW first: x's tile is free again while the MMAs of dx still read D's
        if (want_dw) {
          const bool first = it % kDwTiles == 0;
          if (first) ok = mbar_wait_idle(dw_room, ((it / kDwTiles) & 1) ^ 1, kCodeMma);
          if (!ok) break;
          tcgen05_fence_after();
#pragma unroll 1
          for (int s = 0; s < kNarrowTile / 16; ++s)
            issue_gated<P, kNarrow>(tmem + kDw, d_columns + 128 * s, kDp, x_columns + 128 * s, kXp,
                                    kBf16, true, true, !first || s > 0);
          if (closes_group(t, it)) mma_commit(dw_done);
        }
        mma_commit(x_empty);
        if (want_dx) {
          ok = mbar_wait_idle(dx_room, (it & 1) ^ 1, kCodeMma);
          if (!ok) break;
          tcgen05_fence_after();
#pragma unroll 1
          for (int h = 0; h < 2; ++h)
#pragma unroll 1
            for (int s = 0; 16 * s < p.n; ++s)  // 64 rows of W and columns of D a half
              issue_gated<P, kNarrow>(tmem + kDx, d_rows + h * kXp + 2 * s, kDp,
                                      w_columns + h * 512 + 128 * s, kWp, kBf16, false, true,
                                      h > 0 || s > 0);
          mma_commit(dx_done);
        }
        mma_commit(d_empty);
      }
      // the last arrival lands before the CTA goes away
      if (ok && it > 0) ok = mbar_wait_idle(d_empty, (it - 1) & 1, kCodeMma);
      if (!ok) {  // MMAs in flight finish
        mma_commit(drain);
        mbar_wait(drain, 0, kCodeDrain, kDrainLimitNs);
      }
    }
    __syncwarp();
  } else if (warp >= kRowWarps) {
    give_registers<kGatedProducerRegisters>();
    const int tid = threadIdx.x - kRowWarps * 32;
    uint32_t it = 0, n = 0;
    for (int t = blockIdx.x; t < p.tiles; t += gridDim.x, ++it) {
      if (!mbar_wait_warp(x_empty, (it & 1) ^ 1, kCodeProducer) ||
          !fill_x_tile<T, R>(x_tile, slices, raw_full, raw_empty, t, p, tid, lane, n))
        break;
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(x_full);
    }
  } else {
    take_registers<kRowRegisters>();
    // a thread has a row of p and dx and a row of dW (TMEM lanes 0-63 the gate's, 64-127 the
    // other's), 16 columns of each
    const int quad = warp & 3, c0 = (warp >> 2) * 16, in_tile = quad * 32 + lane;
    const uint32_t at = tmem + (static_cast<uint32_t>(quad * 32) << 16) + c0;
    unsigned char* d_row = d_tile + in_tile * 128;
    constexpr int V = 16 / sizeof(T);
    const T* g = static_cast<const T*>(p.g) + c0;
    T* dx = static_cast<T*>(p.e.out) + c0;
    const int dw_row = (in_tile & (kNarrow - 1)) + (in_tile >= kNarrow ? p.n : 0);
    float* dw = partial + dw_row * p.k + c0;
    const bool dw_some = want_dw && (in_tile & (kNarrow - 1)) < p.n;
    float db[2][16];
#pragma unroll
    for (int i = 0; i < 16; ++i) db[0][i] = db[1][i] = 0.f;
    Pack<T, V> gv[16 / V];
    const auto load_g = [&](int64_t row) {
#pragma unroll
      for (int i = 0; i < 16 / V; ++i) {
        gv[i] = Pack<T, V>{};
        if (row < p.m && c0 + i * V < p.n)
          gv[i] = *reinterpret_cast<const Pack<T, V>*>(g + row * p.n + i * V);
      }
    };
    load_g(static_cast<int64_t>(blockIdx.x) * kNarrowTile + in_tile);
    bool ok = true;
    uint32_t it = 0;
    for (int t = blockIdx.x; ok && t < p.tiles; t += gridDim.x, ++it) {
      const int64_t row = static_cast<int64_t>(t) * kNarrowTile + in_tile;
      ok = mbar_wait_warp(p_done, it & 1, kCodeEpilogue) &&
           mbar_wait_warp(d_empty, (it & 1) ^ 1, kCodeEpilogue);
      if (!ok) break;
      tcgen05_fence_after();
#pragma unroll
      for (int j = 0; j < 16; j += 8) {
        float gate[8], up[8];
        take_p<P>(at + j, gate, up);
        if (j == 8) {
          tcgen05_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(p_room);
        }
        if (c0 + j >= p.n) continue;
        add_bias(gate, bias + c0 + j);
        add_bias(up, bias + kNarrow + c0 + j);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float v = to_float(gv[(j + i) / V].v[(j + i) % V]);
          const float pg = gate[i], pu = up[i];
          // rows past the last have no gradient, but a bias that may be infinite
          gate[i] = row < p.m ? v * pu * activation_slope<ACT>(pg) : 0.f;
          up[i] = row < p.m ? v * activate<ACT>(pg) : 0.f;
          db[0][j + i] += gate[i];
          db[1][j + i] += up[i];
        }
        unsigned char* to = d_row + ((((c0 + j) / 8) ^ (in_tile & 7)) << 4);
        store_d<T>(to, gate);
        store_d<T>(to + kGatedBlock, up);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(d_full);
      // on their way while the MMAs run: the next tile's g, and what dW is so far
      load_g(row + static_cast<int64_t>(gridDim.x) * kNarrowTile);
      if (want_dw && closes_group(t, it)) {
        float4 old[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          old[i] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (dw_some && it >= kDwTiles && c0 + 4 * i < p.k)
            old[i] = *reinterpret_cast<const float4*>(dw + 4 * i);
        }
        ok = mbar_wait_warp(dw_done, (it / kDwTiles) & 1, kCodeEpilogue);
        if (!ok) break;
        tcgen05_fence_after();
        float sum[16];
        take_product<P>(at + kDw, sum);
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(dw_room);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (dw_some && c0 + 4 * i < p.k)
            *reinterpret_cast<float4*>(dw + 4 * i) =
                make_float4(old[i].x + sum[4 * i], old[i].y + sum[4 * i + 1],
                            old[i].z + sum[4 * i + 2], old[i].w + sum[4 * i + 3]);
      }
      if (want_dx) {
        ok = mbar_wait_warp(dx_done, it & 1, kCodeEpilogue);
        if (!ok) break;
        tcgen05_fence_after();
        float sum[16];
        take_product<P>(at + kDx, sum);
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(dx_room);
        if (row < p.m && c0 < p.k) store_columns(dx + row * p.k, sum, p.k - c0, p.e.vec);
      }
    }
    // db: over the lanes, then (below) over the four quads in order.  Every slice was read
    // long ago where all went well; elsewhere nothing is used.
    if (ok) {
      float* sums = reinterpret_cast<float*>(slices) + warp * 32;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float v = db[h][i];
#pragma unroll
          for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
          if (lane == 0) sums[h * 16 + i] = v;
        }
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 0) {
    tcgen05_fence_after();
    tmem_free(tmem, kColumns);
  }
  if (want_dw && threadIdx.x < kGatedRows) {
    const int h = threadIdx.x >> 6, c = threadIdx.x & (kNarrow - 1);
    const float* sums = reinterpret_cast<const float*>(slices);
    if (c < p.n) {
      float total = 0.f;
      for (int q = 0; q < 4; ++q) total += sums[((c >> 4) * 4 + q) * 32 + h * 16 + (c & 15)];
      partial[wide * p.k + h * p.n + c] = total;
    }
  }
}

}  // namespace ictc
