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
// A float32 p has two sums in TMEM, of a1 b1 and of the five other partial products (256
// columns); dx and dW have three, by order (192 each).  dW sums two tiles there, because the
// tensor core truncates when it adds, and is moved into registers.
//
// 1,048,576 x 64 x 64 with SiLU: float32 forward 141 us (3.8 TB/s of x and y), backward 409 us;
// bf16 62 us (4.3 TB/s) and 181 us.
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
  float near;      // backward: what p may be off by, of |x|_2 |w|_2
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

// Eight columns, with three parts the leading sums and, `others` columns on, the others.
template <int P>
__device__ __forceinline__ void take8(uint32_t at, uint32_t others, float2 (&v)[4]) {
  float w[8];
  tmem_load8(at, w);
  if constexpr (P == 3) {
    float y[8];
    tmem_load8(at + others, y);
    tmem_load_wait();
#pragma unroll
    for (int i = 0; i < 4; ++i)  // join_parts
      v[i] = __fadd2_rn(make_float2(w[2 * i], w[2 * i + 1]),
                        make_float2(fmaxf(y[2 * i], -3.402823466e38f),
                                    fmaxf(y[2 * i + 1], -3.402823466e38f)));
  } else {
    tmem_load_wait();
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = make_float2(w[2 * i], w[2 * i + 1]);
  }
}

// act and act' of two values.  f32x2 arithmetic: the row warps are bound by their issue slots.
template <int ACT>
__device__ __forceinline__ void gate_pair(float2 p, float2* a, float2* slope) {
  if constexpr (ACT == ICTC_ACT_SILU) {
    const float2 e = __fmul2_rn(p, make_float2(-1.4426950408889634f, -1.4426950408889634f));
    float2 s;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(s.x) : "f"(e.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(s.y) : "f"(e.y));
    s = __fadd2_rn(s, make_float2(1.f, 1.f));
    s = make_float2(fast_reciprocal(s.x), fast_reciprocal(s.y));
    *a = __fmul2_rn(p, s);
    // s (1 + p (1 - s)) = s + p s (1 - s)
    *slope = __ffma2_rn(*a, __ffma2_rn(s, make_float2(-1.f, -1.f), make_float2(1.f, 1.f)), s);
  } else {
    *a = make_float2(activate<ACT>(p.x), activate<ACT>(p.y));
    *slope = make_float2(activation_slope<ACT>(p.x), activation_slope<ACT>(p.y));
  }
}

// Where 16 bytes of column `col` of a row lie in swizzled boxes of 128 bytes x 128 rows.
template <typename T>
__device__ __forceinline__ uint32_t boxed(int row, int col) {
  constexpr int kWidth = 128 / sizeof(T), V = 16 / sizeof(T);
  return (col / kWidth) * kGatedBlock + swizzled(row, (col % kWidth) / V);
}

// Eight columns of a row to such boxes.
template <typename T>
__device__ __forceinline__ void store_boxed(unsigned char* boxes, int row, int col,
                                            const float2 (&v)[4]) {
  constexpr int V = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 8; i += V) {
    Pack<T, V> o;
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      o.v[j] = from_float<T>(v[(i + j) / 2].x);
      o.v[j + 1] = from_float<T>(v[(i + j) / 2].y);
    }
    *reinterpret_cast<Pack<T, V>*>(boxes + boxed<T>(row, col + i)) = o;
  }
}

struct alignas(64) GatedNarrowMaps {
  CUtensorMap x, g, out;  // boxes of 128 bytes x 128 rows, swizzled; out is y or dx
};

// Warps that take rows out of TMEM.  So many hide its latency and that of the exponentials
// (with eight, bf16 1,048,576 x 64 x 64 forward 127 us, backward 482).
constexpr int kRowWarps = 16;

template <typename T, int THREADS>
__device__ __forceinline__ void stage_bias(float* to, const GatedNarrowArgs& p) {
  for (int i = threadIdx.x; i < kGatedRows; i += THREADS) {
    const int c = i & (kNarrow - 1);
    to[i] = p.bias && c < p.n
                ? to_float(static_cast<const T*>(p.bias)[(i >= kNarrow ? p.n : 0) + c])
                : 0.f;
  }
}

// Eight values of the staged bias.
__device__ __forceinline__ void add_bias(float2 (&v)[4], const float* bias) {
  const float4 a = *reinterpret_cast<const float4*>(bias);
  const float4 b = *reinterpret_cast<const float4*>(bias + 4);
  v[0] = __fadd2_rn(v[0], make_float2(a.x, a.y));
  v[1] = __fadd2_rn(v[1], make_float2(a.z, a.w));
  v[2] = __fadd2_rn(v[2], make_float2(b.x, b.y));
  v[3] = __fadd2_rn(v[3], make_float2(b.z, b.w));
}

// One thread: what the row warps staged leaves for memory, tile after tile.  `groups` of them
// take tiles in turn, and each has a barrier that tells when its tile's boxes were read.
template <typename T, int BUFFERS, int GROUPS>
__device__ __forceinline__ void send_tiles(const unsigned char* boxes, const CUtensorMap* map,
                                           int width, uint64_t* staged, uint64_t* stage_free,
                                           int tiles) {
  uint32_t it = 0;
  for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++it) {
    const uint32_t b = it % BUFFERS;
    if (!mbar_wait_idle(&staged[b], (it / BUFFERS) & 1, kCodeProducer)) break;
    for (int c = 0; c < width; c += 128 / static_cast<int>(sizeof(T)))
      tma_store_2d(boxes + b * kGatedBlock + boxed<T>(0, c), map, c, t * kNarrowTile);
    tma_store_wait_read();
    mbar_arrive(&stage_free[it % GROUPS]);
  }
}

// ------------------------------------------------------------------------- forward

// Row warps, eight producers that cut float32 x (16-bit x arrives as the MMA reads it), and
// the MMA, load and store warps.
constexpr int kGatedProducerWarps = 8;
constexpr int kForwardMmaWarp = kRowWarps + kGatedProducerWarps, kForwardLoadWarp = kForwardMmaWarp + 1,
              kForwardStoreWarp = kForwardMmaWarp + 2;
constexpr int kGatedForwardThreads = 28 * 32;
constexpr int kGatedForwardSlices = 6;
template <typename T>
constexpr int kLeaving = kCut<T> == 3 ? 1 : 2;  // buffers of y
template <typename T>
constexpr size_t kGatedForwardSmem =
    1024 + 3 * kGatedOperand<T> + 2 * kGatedBlock +
    (kCut<T> == 3 ? kGatedForwardSlices * kSliceX<T> : 0) + kGatedRows * 4 + 256;

template <typename T, int ACT>
__global__ void __launch_bounds__(kGatedForwardThreads, 1)
    gated_narrow_forward_kernel(const __grid_constant__ GatedNarrowMaps maps,
                                const __grid_constant__ GatedNarrowArgs p) {
  constexpr int P = kCut<T>, R = kGatedForwardSlices;
  constexpr bool kWide = P == 3;
  constexpr uint32_t kSet = (kWide ? 2 : 1) * kGatedRows;
  extern __shared__ unsigned char raw_smem[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t{1023});
  unsigned char* weights = smem;
  unsigned char* tiles = weights + kGatedOperand<T>;
  unsigned char* leaving = tiles + 2 * kGatedOperand<T>;
  unsigned char* slices = leaving + 2 * kGatedBlock;  // float32
  float* bias = reinterpret_cast<float*>(slices + (kWide ? R * kSliceX<T> : 0));
  uint64_t* raw_full = reinterpret_cast<uint64_t*>(bias + kGatedRows);
  uint64_t* raw_empty = raw_full + R;
  uint64_t* full = raw_empty + R;
  uint64_t* empty = full + 2;
  uint64_t* done = empty + 2;
  uint64_t* room = done + 2;
  uint64_t* staged = room + 2;
  uint64_t* stage_free = staged + 2;
  uint64_t* drain = stage_free + 2;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(drain + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < R; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], kGatedProducerWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&full[i], kWide ? kGatedProducerWarps : 1);
      mbar_init(&empty[i], 1);
      mbar_init(&done[i], 1);
      mbar_init(&room[i], kRowWarps / 2);
      mbar_init(&staged[i], kRowWarps / 2);
      mbar_init(&stage_free[i], 1);
    }
    mbar_init(drain, 1);
    fence_mbarrier_init();
  }
  if (warp == 0) tmem_alloc(tmem_at, 2 * kSet);
  load_gated_weights<T, kGatedForwardThreads>(weights, p);
  stage_bias<T, kGatedForwardThreads>(bias, p);
  fence_proxy_async();
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = *tmem_at;
  const int first = static_cast<int>(blockIdx.x), step = static_cast<int>(gridDim.x);

  if (warp == kForwardLoadWarp) {
    if (lane == 0) {
      bool ok = true;
      if constexpr (kWide) {
        const T* x = static_cast<const T*>(p.x);
        SliceWalk at{first, 0, p.tiles, step, p.m};
        for (uint32_t n = 0; !at.done(); at.next(), ++n) {
          const int slot = n % R;
          ok = mbar_wait_idle(&raw_empty[slot], ((n / R) & 1) ^ 1, kCodeProducer);
          if (!ok) break;
          const uint32_t bytes = slice_bytes<T>(p.k, at.rows());
          mbar_arrive_expect_tx(&raw_full[slot], bytes);
          bulk_g2s(slices + slot * kSliceX<T>, x + at.row() * p.k, bytes, &raw_full[slot]);
        }
      } else {
        uint32_t it = 0;
        for (int t = first; t < p.tiles; t += step, ++it) {
          const int s = it & 1;
          ok = mbar_wait_idle(&empty[s], ((it >> 1) & 1) ^ 1, kCodeProducer);
          if (!ok) break;
          mbar_arrive_expect_tx(&full[s], kGatedBlock);
          tma_load_2d(tiles + s * kGatedBlock, &maps.x, 0, t * kNarrowTile, &full[s]);
        }
      }
      if (!ok) settle_copies();
    }
    __syncwarp();
  } else if (warp == kForwardStoreWarp) {
    if (lane == 0)
      send_tiles<T, kLeaving<T>, 2>(leaving, &maps.out, p.n, staged, stage_free, p.tiles);
    __syncwarp();
  } else if (warp == kForwardMmaWarp) {
    if (lane == 0) {
      bool ok = true;
      uint32_t it = 0;
      for (int t = first; t < p.tiles; t += step, ++it) {
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
  } else if (kWide && warp >= kRowWarps && warp < kForwardMmaWarp) {
    const int tid = threadIdx.x - kRowWarps * 32, unit = tid & 15, r0 = tid >> 4;
    const int columns = (p.k + 15) & ~15;  // that the MMAs read
    uint32_t it = 0, n = 0;                // tiles and slices so far
    bool ok = true;
    for (int t = first; ok && t < p.tiles; t += step, ++it) {
      const int s = it & 1;
      ok = mbar_wait_warp(&empty[s], ((it >> 1) & 1) ^ 1, kCodeProducer);
      unsigned char* tile = tiles + s * kGatedOperand<T>;
      SliceWalk at{t, 0, p.tiles, step, p.m};
#pragma unroll 1
      for (int q = 0; ok && q < kNarrowTile / kSliceRows; ++q, ++at.slice) {
        Slice<T> slice{nullptr, nullptr, p.k, 0, 0};
        const bool some = at.row() < p.m;
        const int slot = n % R;
        if (some) {
          ok = mbar_wait_warp(&raw_full[slot], (n / R) & 1, kCodeProducer);
          if (!ok) break;
          slice.raw = reinterpret_cast<const T*>(slices + slot * kSliceX<T>);
          slice.rows = at.rows();
        }
        float v[2][4];
        uint32_t seen = 0;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          read_unit<true>(slice, r0 + 16 * j, unit, v[j]);
          seen |= unit_bits<true>(v[j]);
        }
        if (4 * unit < columns)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            store_unit<T>(tile, kGatedBlock, q * kSliceRows + r0 + 16 * j, unit, v[j]);
        if (some) {
          release_slot(&raw_empty[slot], seen, lane);
          ++n;
        }
      }
      if (!ok) break;
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[s]);
    }
  } else if (warp < kRowWarps) {
    // eight warps for each of the two sets, every other tile: rows of a quad, half the columns
    const int quad = warp & 3, half = (warp >> 2) & 1, s = warp >> 3;
    constexpr int L = kLeaving<T>;
    uint32_t it = 0;
    for (int t = first + s * step; t < p.tiles; t += 2 * step, ++it) {
      const uint32_t tile = 2 * it + s;  // of the CTA's
      unsigned char* boxes = leaving + (tile % L) * kGatedBlock;
      // the boxes were last those of tile - L.  One barrier for both groups would not do: a
      // group can come back two tiles later, when its phase looks like the one before.
      const uint32_t last = tile + 2 - L;  // + 2, which keeps parities
      if (!mbar_wait_warp(&done[s], it & 1, kCodeEpilogue) ||
          !mbar_wait_warp(&stage_free[last & 1], ((last >> 1) & 1) ^ 1, kCodeEpilogue))
        break;
      tcgen05_fence_after();
      const uint32_t at = tmem + s * kSet + (static_cast<uint32_t>(quad * 32) << 16) + half * 32;
#pragma unroll
      for (int j = 0; j < 32; j += 8) {
        const int col = half * 32 + j;
        float2 gate[4], up[4];
        take8<P>(at + j, kGatedRows, gate);
        take8<P>(at + kNarrow + j, kGatedRows, up);
        if (j == 24) {
          tcgen05_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&room[s]);
        }
        add_bias(gate, bias + col);
        add_bias(up, bias + kNarrow + col);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float2 a, slope;
          gate_pair<ACT>(gate[i], &a, &slope);
          up[i] = __fmul2_rn(up[i], a);
        }
        store_boxed<T>(boxes, quad * 32 + lane, col, up);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&staged[tile % L]);
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
//
// A tile's chain is p, D, then dW and dx (their MMAs in turn: two that add to the same sums
// take 110 to 160 cycles each, to different ones 76), then dx out.  16-bit types have room to
// overlap two tiles of it: p of the next is formed while D of one waits for its products.  In
// float32 one tile fills shared memory and TMEM: g lands where D's third parts will be, dx
// leaves from where its first parts were, dx's sums lie where p's were, and the row warps cut
// the next x while the tensor cores work on D.

constexpr int kRowThreads = kRowWarps * 32;
constexpr int kBackMmaWarp = kRowWarps, kBackLoadWarp = kRowWarps + 1,
              kBackStoreWarp = kRowWarps + 2;
constexpr int kBackThreads = 20 * 32;
// Registers move to the row warps, which hold sums of dW and db.
constexpr int kBackLaunchRegisters = 96;  // 65,536 / 640, in steps of 8
constexpr int kRowRegisters = 104, kIssueRegisters = 64;
static_assert(kRowWarps * kRowRegisters + 4 * kIssueRegisters <= 20 * kBackLaunchRegisters);

template <typename T>
constexpr int kBackBuffers = kCut<T> == 3 ? 1 : 2;  // of x, D, and (16-bit) g and p
// Bytes of the raw x tile, or of two g tiles and the dx that leaves
template <typename T>
constexpr uint32_t kBackMore = kCut<T> == 3 ? kNarrowTile * kNarrow * 4 : 3 * kGatedBlock;
template <typename T>
constexpr size_t kGatedBackwardSmem =
    1024 + (1 + 3 * kBackBuffers<T>)*kGatedOperand<T> + kBackMore<T> + kGatedRows * 4 + 512;

// Eight columns of D to their tile, part by part.
template <typename T>
__device__ __forceinline__ void store_d(unsigned char* at, const float2 (&v)[4]) {
  if constexpr (kCut<T> == 3) {
    uint32_t part[4][3];
#pragma unroll
    for (int j = 0; j < 4; ++j) cut_pair(v[j].x, v[j].y, part[j]);
#pragma unroll
    for (int q = 0; q < 3; ++q)
      *reinterpret_cast<uint4*>(at + q * 2 * kGatedBlock) =
          make_uint4(part[0][q], part[1][q], part[2][q], part[3][q]);
  } else {
    Pack<T, 8> o;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      o.v[2 * j] = from_float<T>(v[j].x);
      o.v[2 * j + 1] = from_float<T>(v[j].y);
    }
    *reinterpret_cast<Pack<T, 8>*>(at) = o;
  }
}

// One K step of a 64-column product: with three parts a1 (b1 | b2 | b3), a2 (b1 | b2), a3 b1
// into sums of order 0, 1 and 2.
template <int P>
__device__ __forceinline__ void issue_orders(uint32_t d, uint64_t a, uint64_t a_part, uint64_t b,
                                             bool bf16, bool a_mn, bool b_mn, bool add) {
  const uint32_t one = mma_descriptor(bf16, a_mn, b_mn, kNarrowTile, kNarrow);
  if constexpr (P == 3) {
    mma_f16(d, a, b, mma_descriptor(bf16, a_mn, b_mn, kNarrowTile, 3 * kNarrow), add);
    mma_f16(d + kNarrow, a + a_part, b,
            mma_descriptor(bf16, a_mn, b_mn, kNarrowTile, 2 * kNarrow), true);
    mma_f16(d + 2 * kNarrow, a + 2 * a_part, b, one, true);
  } else {
    mma_f16(d, a, b, one, add);
  }
}

// Eight columns of such a product.
template <int P>
__device__ __forceinline__ void take_orders(uint32_t at, float2 (&v)[4]) {
  float w[8];
  tmem_load8(at, w);
  if constexpr (P == 3) {
    float y[8], z[8];
    tmem_load8(at + kNarrow, y);
    tmem_load8(at + 2 * kNarrow, z);
    tmem_load_wait();
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = join_parts(w[i], y[i] + z[i]);
  } else {
    tmem_load_wait();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = make_float2(w[2 * i], w[2 * i + 1]);
}

// Relu in float32: gate projections within the bounds of their error are computed again, in the
// order of k and the bias last, so that the slope is that of every other path.  |x|_2 |w|_2
// bounds a row's sums; a lane adds up those of its row (2 elements in 10^5 as a rule) from the
// parts in shared memory.  1,048,576 x 64 x 64 backward: 445 us, without it 404; with whole
// numbers for operands, where one in 14 is 0, some 2.4 times that.

// Whether a p that may be off by `error` may have another sign.  Rows and columns of zeros have
// no error, those with an infinity no p of a finite value.
__device__ __forceinline__ bool is_near(float p, float error) {
  return error > 0.f && error <= 3.402823466e38f && fabsf(p) <= error;
}

// At least |x_r|_2 of a row of the x tile, from its leading parts: bf16 sums of 32 squares each
// of the two halves, low by less than the fifth that is added.  Where squares leave the range,
// |x_r|_1.
__device__ __forceinline__ float row_size(const unsigned char* row, int lane) {
  __nv_bfloat162 squares = __floats2bfloat162_rn(0.f, 0.f);
  const auto block = [&](int i) {  // another one in each lane: their banks differ
    return *reinterpret_cast<const uint4*>(row + (((i + lane) & 7) << 4));
  };
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint4 q = block(i);
    const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(&u[j]);
      squares = __hfma2(v, v, squares);
    }
  }
  const float sum = 1.2f * (__low2float(squares) + __high2float(squares));
  if (sum > 1e-30f && sum < 1e38f) return sum * rsqrtf(sum);
  float size = 0.f;
#pragma unroll 1
  for (int i = 0; i < 8; ++i) {
    const uint4 q = block(i);
    const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      size += __uint_as_float(u[j] << 16 & 0x7fffffffu) + __uint_as_float(u[j] & 0x7fff0000u);
  }
  return 1.2f * size;
}

// |w|_2 of the gate's rows.  Whole warps, at the kernel's start.
template <int THREADS>
__device__ __forceinline__ void stage_gate_sizes(float* to, const GatedNarrowArgs& p) {
  const int lane = threadIdx.x & 31;
  for (int c = threadIdx.x >> 5; c < p.n; c += THREADS / 32) {
    const float* row = static_cast<const float*>(p.w) + c * p.ldw;
    double sum = 0.0;
    for (int i = lane; i < p.k; i += 32) sum = fma(static_cast<double>(row[i]), static_cast<double>(row[i]), sum);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) to[c] = 1.001f * static_cast<float>(sqrt(sum));
  }
}

// Four values of a row from the parts of an operand, exactly.
__device__ __forceinline__ void join_unit(const unsigned char* operand, int row, int unit,
                                          float (&v)[4]) {
  const unsigned char* at = operand + swizzled(row, unit >> 1) + (unit & 1) * 8;
  float part[3][4];
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    const uint2 u = *reinterpret_cast<const uint2*>(at + q * kGatedBlock);
    part[q][0] = __uint_as_float(u.x << 16);
    part[q][1] = __uint_as_float(u.x & 0xffff0000u);
    part[q][2] = __uint_as_float(u.y << 16);
    part[q][3] = __uint_as_float(u.y & 0xffff0000u);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = part[0][j] + (part[1][j] + part[2][j]);
}

// Whole warp: the gate projections of the columns `col` to col + 7 of a row a lane; those of a
// row may be off by `near` times a column's size (0: no row).
__device__ __forceinline__ void settle_gate(float2 (&gate)[4], float near, float most,
                                            const float* sizes, const float* bias,
                                            const unsigned char* x, const unsigned char* w, int n,
                                            int k, int row, int col) {
  if (col >= n) return;
  const auto least = [](float2 a, float2 b) {
    return fminf(fminf(fabsf(a.x), fabsf(a.y)), fminf(fabsf(b.x), fabsf(b.y)));
  };
  float low = least(gate[0], gate[1]);
  if (col + 4 < n) low = fminf(low, least(gate[2], gate[3]));  // n is a multiple of 4
  if (!__any_sync(0xffffffffu, is_near(low, near * most))) return;
  uint32_t mine = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = i % 2 ? gate[i / 2].y : gate[i / 2].x;
    if (col + i < n && is_near(v, near * sizes[col + i])) mine |= 1u << i;
  }
#pragma unroll 1
  for (; mine != 0; mine &= mine - 1) {
    const int i = __ffs(mine) - 1;
    float sum = 0.f;
#pragma unroll 1
    for (int u = 0; 4 * u < k; ++u) {
      float a[4], b[4];
      join_unit(x, row, u, a);
      join_unit(w, col + i, u, b);
#pragma unroll
      for (int j = 0; j < 4; ++j) sum = fmaf(a[j], b[j], sum);
    }
    sum += bias[col + i];
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (q == i) (q % 2 ? gate[q / 2].y : gate[q / 2].x) = sum;
  }
  __syncwarp();
}

template <typename T, int ACT>
__global__ void __launch_bounds__(kBackThreads, 1)
    gated_narrow_backward_kernel(const __grid_constant__ GatedNarrowMaps maps,
                                 const __grid_constant__ GatedNarrowArgs p) {
  constexpr int P = kCut<T>, B = kBackBuffers<T>, kLag = B - 1;
  constexpr bool kWide = P == 3;
  constexpr bool kSettles = kWide && ACT == ICTC_ACT_RELU;
  constexpr uint32_t kPset = kWide ? 0 : kGatedRows;  // TMEM columns from one p to the next
  constexpr uint32_t kDx = kWide ? 0 : 2 * kGatedRows, kDxSet = kWide ? 0 : kNarrow;
  constexpr uint32_t kDw = kWide ? 2 * kGatedRows : 2 * kGatedRows + 2 * kNarrow;
  extern __shared__ unsigned char raw_smem[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t{1023});
  unsigned char* weights = smem;
  unsigned char* x_tiles = weights + kGatedOperand<T>;
  unsigned char* d_tiles = x_tiles + B * kGatedOperand<T>;  // [parts][gate, up][128 rows][64]
  unsigned char* more = d_tiles + 2 * B * kGatedOperand<T>;
  unsigned char* g_tiles = kWide ? d_tiles + 4 * kGatedBlock : more;
  unsigned char* leaving = kWide ? d_tiles : more + 2 * kGatedBlock;
  float* bias = reinterpret_cast<float*>(more + kBackMore<T>);
  float* sizes = bias + kGatedRows;  // of the gate's rows
  uint64_t* raw_full = reinterpret_cast<uint64_t*>(sizes + kNarrow);
  uint64_t* raw_empty = raw_full + 1;
  uint64_t* x_full = raw_empty + 1;
  uint64_t* x_empty = x_full + B;
  uint64_t* g_full = x_empty + B;
  uint64_t* g_read = g_full + B;
  uint64_t* p_done = g_read + B;
  uint64_t* p_room = p_done + B;
  uint64_t* d_full = p_room + B;
  uint64_t* d_empty = d_full + B;
  uint64_t* dx_done = d_empty + B;
  uint64_t* dx_room = dx_done + B;
  uint64_t* dw_done = dx_room + B;
  uint64_t* dw_room = dw_done + 1;
  uint64_t* staged = dw_room + 1;
  uint64_t* stage_free = staged + 1;
  uint64_t* drain = stage_free + 1;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(drain + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(raw_full, 1);
    mbar_init(raw_empty, kRowWarps);
    for (int i = 0; i < B; ++i) {
      mbar_init(&x_full[i], kWide ? kRowWarps : 1);
      mbar_init(&x_empty[i], 1);
      mbar_init(&g_full[i], 1);
      mbar_init(&g_read[i], kRowWarps);
      mbar_init(&p_done[i], 1);
      mbar_init(&p_room[i], kRowWarps);
      mbar_init(&d_full[i], kRowWarps);
      mbar_init(&d_empty[i], 1);
      mbar_init(&dx_done[i], 1);
      mbar_init(&dx_room[i], kRowWarps);
    }
    mbar_init(dw_done, 1);
    mbar_init(dw_room, kRowWarps);
    mbar_init(staged, kRowWarps);
    mbar_init(stage_free, 1);
    mbar_init(drain, 1);
    fence_mbarrier_init();
  }
  if (warp == 0) tmem_alloc(tmem_at, 512);
  load_gated_weights<T, kBackThreads>(weights, p);
  stage_bias<T, kBackThreads>(bias, p);
  if constexpr (kSettles) stage_gate_sizes<kBackThreads>(sizes, p);
  // columns of x past k and of D past n may never be written, but the MMAs read them
  for (uint32_t i = threadIdx.x; i < 3 * B * kGatedOperand<T> / 16; i += kBackThreads)
    reinterpret_cast<uint4*>(x_tiles)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async();
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = *tmem_at;
  const bool want_dx = p.e.out != nullptr, want_dw = p.partial != nullptr;
  const int step = static_cast<int>(gridDim.x), first = static_cast<int>(blockIdx.x);
  const auto closes_group = [&](int t, uint32_t it) {
    return it % kDwTiles == kDwTiles - 1 || t + step >= p.tiles;
  };
  const int wide = 2 * p.n;
  float* partial =
      want_dw ? p.partial + static_cast<int64_t>(first) * (wide * p.k + wide) : nullptr;

  if (warp >= kRowWarps) {
    give_registers<kIssueRegisters>();
    if (warp == kBackLoadWarp && lane == 0) {
      bool ok = true;
      uint32_t it = 0;
      for (int t = first; t < p.tiles; t += step, ++it) {
        const uint32_t b = it & kLag, phase = (it >> kLag) & 1;
        const int64_t row0 = static_cast<int64_t>(t) * kNarrowTile;
        if constexpr (kWide) {
          ok = mbar_wait_idle(raw_empty, phase ^ 1, kCodeProducer);
          if (!ok) break;
          const int64_t left = p.m - row0;
          const uint32_t bytes =
              static_cast<uint32_t>(left < kNarrowTile ? left : kNarrowTile) * p.k * 4;
          mbar_arrive_expect_tx(raw_full, bytes);
          bulk_g2s(more, static_cast<const float*>(p.x) + row0 * p.k, bytes, raw_full);
          ok = mbar_wait_idle(&d_empty[0], phase ^ 1, kCodeProducer);
        } else {
          ok = mbar_wait_idle(&x_empty[b], phase ^ 1, kCodeProducer);
          if (!ok) break;
          mbar_arrive_expect_tx(&x_full[b], kGatedBlock);
          tma_load_2d(x_tiles + b * kGatedBlock, &maps.x, 0, static_cast<int>(row0), &x_full[b]);
          ok = mbar_wait_idle(&g_read[b], phase ^ 1, kCodeProducer);
        }
        if (!ok) break;
        mbar_arrive_expect_tx(&g_full[b], kNarrowTile * kNarrow * sizeof(T));
        for (int c = 0; c < kNarrow; c += 128 / static_cast<int>(sizeof(T)))
          tma_load_2d(g_tiles + b * kGatedBlock + boxed<T>(0, c), &maps.g, c,
                      static_cast<int>(row0), &g_full[b]);
      }
      if (!ok) settle_copies();
    }
    if (warp == kBackStoreWarp && lane == 0 && want_dx)
      send_tiles<T, 1, 1>(leaving, &maps.out, p.k, staged, stage_free, p.tiles);
    if (warp == kBackMmaWarp && lane == 0) {
      constexpr bool kBf16 = !std::is_same_v<T, __half>;
      const uint32_t wa = smem_addr(weights);
      // MN-major with the parts behind one another as further columns
      const uint64_t w_columns = matrix_descriptor(wa, kGatedRows * 128, 1024);
      constexpr uint64_t kXp = kGatedBlock / 16, kDp = 2 * kXp;
      const int steps = (p.n + 15) / 16, dx_steps = want_dx ? 2 * steps : 0;
      const int dw_steps = want_dw ? kNarrowTile / 16 : 0;
      bool ok = true;
      uint32_t it = 0;
      const auto form_p = [&](uint32_t i) {
        const uint32_t b = i & kLag, phase = (i >> kLag) & 1;
        ok = mbar_wait_idle(&x_full[b], phase, kCodeMma);
        if (ok && (!kWide || want_dx))  // in float32 dx's sums lie where p will be
          ok = mbar_wait_idle(kWide ? &dx_room[b] : &p_room[b], phase ^ 1, kCodeMma);
        if (!ok) return;
        tcgen05_fence_after();
        issue_p<T>(tmem + b * kPset, smem_addr(x_tiles + b * kGatedOperand<T>), wa, p.k);
        mma_commit(&p_done[b]);
      };
      if (kLag && first < p.tiles) form_p(0);
      for (int t = first; ok && t < p.tiles; t += step, ++it) {
        const uint32_t b = it & kLag, phase = (it >> kLag) & 1;
        if (!kLag) form_p(it);
        else if (t + step < p.tiles) form_p(it + 1);
        if (ok) ok = mbar_wait_idle(&d_full[b], phase, kCodeMma);
        if (!ok) break;
        const bool opens = it % kDwTiles == 0;
        if (want_dw && opens)
          ok = mbar_wait_idle(dw_room, ((it / kDwTiles) & 1) ^ 1, kCodeMma);
        if (ok && !kWide && want_dx) ok = mbar_wait_idle(&dx_room[b], phase ^ 1, kCodeMma);
        if (!ok) break;
        tcgen05_fence_after();
        const uint32_t xa = smem_addr(x_tiles + b * kGatedOperand<T>);
        const uint32_t da = smem_addr(d_tiles + b * 2 * kGatedOperand<T>);
        const uint64_t x_columns = matrix_descriptor(xa, kGatedBlock, 1024);
        const uint64_t d_rows = matrix_descriptor(da, 0, 1024);               // K-major
        const uint64_t d_columns = matrix_descriptor(da, kGatedBlock, 1024);  // two blocks
        const auto add_dx = [&](int s) {  // 64 columns of D and rows of W a half
          const int h = s >= steps, q = s - h * steps;
          issue_orders<P>(tmem + kDx + b * kDxSet, d_rows + h * kXp + 2 * q, kDp,
                          w_columns + h * 512 + 128 * q, kBf16, false, true, s > 0);
        };
        // x is free after dW: the last steps of dx run while it is filled again
        int s = 0;
#pragma unroll 1
        for (int i = 0; i < dw_steps; ++i) {
          issue_orders<P>(tmem + kDw, d_columns + 128 * i, kDp, x_columns + 128 * i, kBf16, true,
                          true, !opens || i > 0);
          if ((!kWide || i % 2 == 1) && s < dx_steps) add_dx(s++);
        }
        mma_commit(&x_empty[b]);
#pragma unroll 1
        for (; s < dx_steps; ++s) add_dx(s);
        if (want_dw && closes_group(t, it)) mma_commit(dw_done);
        if (want_dx) mma_commit(&dx_done[b]);
        mma_commit(&d_empty[b]);
      }
      // the last arrival lands before the CTA goes away
      if (ok && it > 0)
        ok = mbar_wait_idle(&d_empty[(it - 1) & kLag], ((it - 1) >> kLag) & 1, kCodeMma);
      if (!ok) {  // MMAs in flight finish
        mma_commit(drain);
        mbar_wait(drain, 0, kCodeDrain, kDrainLimitNs);
      }
    }
    __syncwarp();
  } else {
    take_registers<kRowRegisters>();
    // a thread has a row of p and dx and a row of dW (TMEM lanes 0-63 the gate's, 64-127 the
    // other's), 16 columns of each
    constexpr int V = 16 / sizeof(T);
    const int quad = warp & 3, c0 = (warp >> 2) * 16, in_tile = quad * 32 + lane;
    const uint32_t at = tmem + (static_cast<uint32_t>(quad * 32) << 16) + c0;
    float2 db[2][8], dw[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) db[0][i] = db[1][i] = dw[i] = make_float2(0.f, 0.f);
    bool ok = true;
    float most = 0.f;  // of the gate's sizes
    if constexpr (kSettles)
      for (int c = 0; c < p.n; ++c) most = fmaxf(most, sizes[c]);

    // float32: the next tile's x, cut
    const auto fill_x = [&](int t, uint32_t it) {
      if constexpr (kWide) {
        ok = mbar_wait_warp(raw_full, it & 1, kCodeProducer) &&
             mbar_wait_warp(&x_empty[0], (it & 1) ^ 1, kCodeProducer);
        if (!ok) return;
        const int unit = threadIdx.x & 15, r0 = threadIdx.x >> 4;
        const int64_t left = p.m - static_cast<int64_t>(t) * kNarrowTile;
        const Slice<T> raw{reinterpret_cast<const T*>(more), nullptr, p.k,
                           left < kNarrowTile ? static_cast<int>(left) : kNarrowTile, 0};
        float v[4][4];
        uint32_t seen = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          read_unit<true>(raw, r0 + 32 * j, unit, v[j]);
          seen |= unit_bits<true>(v[j]);
        }
        release_slot(raw_empty, seen, lane);
        if (4 * unit < p.k)
#pragma unroll
          for (int j = 0; j < 4; ++j) store_unit<T>(x_tiles, kGatedBlock, r0 + 32 * j, unit, v[j]);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&x_full[0]);
      }
    };

    // what the products of a tile left
    const auto take_tile = [&](int t, uint32_t it) {
      const uint32_t b = it & kLag, phase = (it >> kLag) & 1;
      if (want_dw && closes_group(t, it)) {
        ok = mbar_wait_warp(dw_done, (it / kDwTiles) & 1, kCodeEpilogue);
        if (!ok) return;
        tcgen05_fence_after();
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float2 sum[4];
          take_orders<P>(at + kDw + 8 * j, sum);
#pragma unroll
          for (int i = 0; i < 4; ++i) dw[4 * j + i] = __fadd2_rn(dw[4 * j + i], sum[i]);
        }
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(dw_room);
      }
      if (!want_dx) return;
      ok = mbar_wait_warp(&dx_done[b], phase, kCodeEpilogue);
      if (ok && !kWide) ok = mbar_wait_warp(stage_free, (it & 1) ^ 1, kCodeEpilogue);
      if (!ok) return;
      tcgen05_fence_after();
#pragma unroll
      for (int j = 0; j < 16; j += 8) {
        float2 sum[4];
        take_orders<P>(at + kDx + b * kDxSet + j, sum);
        if (j == 8) {
          tcgen05_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&dx_room[b]);
        }
        store_boxed<T>(leaving, in_tile, c0 + j, sum);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(staged);
    };

    if (kWide && first < p.tiles) fill_x(first, 0);
    uint32_t it = 0;
    for (int t = first; ok && t < p.tiles; t += step, ++it) {
      const uint32_t b = it & kLag, phase = (it >> kLag) & 1;
      const bool in = static_cast<int64_t>(t) * kNarrowTile + in_tile < p.m;
      ok = mbar_wait_warp(&g_full[b], phase, kCodeEpilogue);
      if (!ok) break;
      Pack<T, V> g[16 / V];
      uint32_t seen = 0;
#pragma unroll
      for (int i = 0; i < 16; i += V) {
        uint32_t q[4];
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3])
                     : "r"(smem_addr(g_tiles + b * kGatedBlock + boxed<T>(in_tile, c0 + i)))
                     : "memory");
        g[i / V] = *reinterpret_cast<const Pack<T, V>*>(q);
        seen |= q[0];
      }
      release_slot(&g_read[b], seen, lane);
      float near = 0.f;
      if constexpr (kSettles) {  // while the tensor cores form p
        ok = mbar_wait_warp(&x_full[b], phase, kCodeEpilogue);
        if (!ok) break;
        if (in) near = p.near * row_size(x_tiles + in_tile * 128, lane);
      }
      ok = mbar_wait_warp(&p_done[b], phase, kCodeEpilogue);
      // where D goes: g has been read and dx has left, or the products before last are done
      if (ok && kWide) ok = mbar_wait_warp(&g_read[0], phase, kCodeEpilogue);
      if (ok && kWide && want_dx) ok = mbar_wait_warp(stage_free, phase ^ 1, kCodeEpilogue);
      if (ok && !kWide) ok = mbar_wait_warp(&d_empty[b], phase ^ 1, kCodeEpilogue);
      if (!ok) break;
      tcgen05_fence_after();
      unsigned char* d_row = d_tiles + b * 2 * kGatedOperand<T> + in_tile * 128;
      const bool whole = static_cast<int64_t>(t + 1) * kNarrowTile <= p.m;
#pragma unroll
      for (int j = 0; j < 16; j += 8) {
        float2 gate[4], up[4];
        take8<P>(at + b * kPset + j, kGatedRows, gate);
        take8<P>(at + b * kPset + kNarrow + j, kGatedRows, up);
        if (j == 8) {
          tcgen05_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_room[b]);
        }
        // up to the last K step of dx: zeros past n, over what dx left there
        if (c0 + j >= ((p.n + 15) & ~15)) continue;
        add_bias(gate, bias + c0 + j);
        add_bias(up, bias + kNarrow + c0 + j);
        if constexpr (kSettles)
          settle_gate(gate, near, most, sizes, bias, x_tiles, weights, p.n, p.k, in_tile, c0 + j);
        if (!whole && !in) {  // no gradient past the last row, but a bias that may be infinite
#pragma unroll
          for (int i = 0; i < 4; ++i) gate[i] = up[i] = make_float2(0.f, 0.f);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at_g = j + 2 * i;
          const float2 v = make_float2(to_float(g[at_g / V].v[at_g % V]),
                                       to_float(g[(at_g + 1) / V].v[(at_g + 1) % V]));
          float2 a, slope;
          gate_pair<ACT>(gate[i], &a, &slope);
          gate[i] = __fmul2_rn(__fmul2_rn(v, up[i]), slope);
          up[i] = __fmul2_rn(v, a);
          db[0][j / 2 + i] = __fadd2_rn(db[0][j / 2 + i], gate[i]);
          db[1][j / 2 + i] = __fadd2_rn(db[1][j / 2 + i], up[i]);
        }
        unsigned char* to = d_row + ((((c0 + j) / 8) ^ (in_tile & 7)) << 4);
        store_d<T>(to, gate);
        store_d<T>(to + kGatedBlock, up);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&d_full[b]);
      if (kLag) {
        if (it > 0) take_tile(t - step, it - 1);
      } else {
        if (t + step < p.tiles) fill_x(t + step, it + 1);
        if (ok) take_tile(t, it);
      }
    }
    if (kLag && ok && it > 0)
      take_tile(first + static_cast<int>(it - 1) * step, it - 1);
    if (ok && want_dw) {
      // every product is done: x's tile has room for the sums of db
      float* sums = reinterpret_cast<float*>(x_tiles) + warp * 32;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float v = i % 2 ? db[h][i / 2].y : db[h][i / 2].x;
#pragma unroll
          for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
          if (lane == 0) sums[h * 16 + i] = v;
        }
      const int column = in_tile & (kNarrow - 1);  // of D, in its half
      float* to = partial + ((in_tile >= kNarrow ? p.n : 0) + column) * p.k + c0;
      if (column < p.n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (c0 + 4 * i < p.k)
            *reinterpret_cast<float4*>(to + 4 * i) =
                make_float4(dw[2 * i].x, dw[2 * i].y, dw[2 * i + 1].x, dw[2 * i + 1].y);
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 0) {
    tcgen05_fence_after();
    tmem_free(tmem, 512);
  }
  if (want_dw && threadIdx.x < kGatedRows) {  // db over the four quads, in order
    const int h = threadIdx.x >> 6, c = threadIdx.x & (kNarrow - 1);
    const float* sums = reinterpret_cast<const float*>(x_tiles);
    if (c < p.n) {
      float total = 0.f;
      for (int q = 0; q < 4; ++q) total += sums[((c >> 4) * 4 + q) * 32 + h * 16 + (c & 15)];
      partial[wide * p.k + h * p.n + c] = total;
    }
  }
}

}  // namespace ictc
