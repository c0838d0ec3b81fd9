// Linear layers of at most 64 inputs and 64 outputs over many rows (radial networks over
// edges): forward and the whole backward as one kernel each.
//
// These are bound by HBM, so every operand byte should move once.  W is cut and laid out
// in shared memory once per CTA.  Rows come in tiles of 128; because operands are
// contiguous, 32 rows are one bulk copy whatever their width, and a ring of such slices
// keeps the copies ahead of the arithmetic.  The backward forms d = g act'(p) on the way
// in, sums db from it, and uses the one swizzled copy of each tile in both orders: d as
// the K-major operand of d W and, with the same bytes read as MN-major, of d^T x.
//
//   dx = d W      M = 128 rows, reduction over n <= 64
//   dW = d^T x    M = 64 columns of d (and, as the MMA takes 128, the 64 of x beside
//                 them, whose products are dropped), reduction over the tile's 128 rows
//
// dW stays in registers over all of a CTA's rows: TMEM holds the sums of two tiles at a
// time (the tensor core truncates when it adds), and the CTAs' partial results are
// summed in CTA order.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "dense_epilogue.cuh"
#include "tcgen05.cuh"

namespace ictc {

constexpr int kNarrow = 64;          // most inputs and outputs
constexpr int kNarrowTile = 128;     // rows of a tile
constexpr int kSliceRows = 32;       // rows of a bulk copy
constexpr int kNarrowThreadsL = 512; // 8 epilogue and 8 producer warps
constexpr int kNarrowMmaWarp = 8, kNarrowCopyWarp = 9;  // producer warps with an extra duty
constexpr int kDwTiles = 2;          // tiles whose d^T x is summed in TMEM

template <typename T>
constexpr int kCut = sizeof(T) == 4 ? 3 : 1;  // bf16 parts of an operand value

// Bytes of a slice: x, and for the backward g and p.
template <typename T>
constexpr uint32_t kSliceX = kSliceRows * kNarrow * sizeof(T);
constexpr uint32_t kSliceP = kSliceRows * kNarrow * sizeof(float);

template <typename T>
constexpr uint32_t kNarrowW = kCut<T> * kNarrow * 128;
template <typename T>
constexpr uint32_t kNarrowOperand = kCut<T> * kNarrowTile * 128;

constexpr int kForwardSlices = 8;
template <typename T>
constexpr int kBackwardSlices = sizeof(T) == 4 ? 3 : 4;
constexpr uint32_t kNarrowStaging = 8 * 4096;

template <typename T>
constexpr size_t kNarrowForwardSmem =
    1024 + kNarrowW<T> + 2 * kNarrowOperand<T> + kForwardSlices * kSliceX<T> + kNarrowStaging + 512;
template <typename T>
constexpr uint32_t kBackwardSlice = 2 * kSliceX<T> + kSliceP;
template <typename T>
constexpr size_t kNarrowBackwardSmem = 1024 + kNarrowW<T> + 2 * kNarrowOperand<T> +
                                       kBackwardSlices<T> * kBackwardSlice<T> + kNarrowStaging +
                                       512;

struct NarrowArgs {
  const void *x, *w, *g;   // x [m, k], w [n, k] (rows ldw apart), g [m, n]
  const float* preact;     // [m, n] p
  int64_t m, ldw;
  int n, k, tiles;
  float* partial;          // [gridDim.x][n k + n]: dW, db
  Epilogue e;              // forward: y; backward: dx
};

// Cuts four values and stores them as half of a 16-byte chunk: columns 4 u .. 4 u + 3 of
// row r of a [rows][64] operand (`piece` bytes from one part to the next).
template <typename T>
__device__ __forceinline__ void store_unit(unsigned char* dst, uint32_t piece, int r, int u,
                                           const float (&v)[4]) {
  unsigned char* at = dst + swizzled(r, u >> 1) + (u & 1) * 8;
  if constexpr (kCut<T> == 3) {
    uint32_t part[3][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t u0 = __float_as_uint(v[2 * j]), u1 = __float_as_uint(v[2 * j + 1]);
      part[0][j] = __byte_perm(u0, u1, 0x7632);
      const float r0 = v[2 * j] - __uint_as_float(u0 & 0xffff0000u);
      const float r1 = v[2 * j + 1] - __uint_as_float(u1 & 0xffff0000u);
      const uint32_t v0 = __float_as_uint(r0), v1 = __float_as_uint(r1);
      part[1][j] = __byte_perm(v0, v1, 0x7632);
      const float s0 = r0 - __uint_as_float(v0 & 0xffff0000u);
      const float s1 = r1 - __uint_as_float(v1 & 0xffff0000u);
      part[2][j] = __byte_perm(__float_as_uint(s0), __float_as_uint(s1), 0x7632);
    }
#pragma unroll
    for (int q = 0; q < 3; ++q)
      *reinterpret_cast<uint2*>(at + q * piece) = make_uint2(part[q][0], part[q][1]);
  } else {
    Pack<T, 4> o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o.v[j] = from_float<T>(v[j]);
    *reinterpret_cast<Pack<T, 4>*>(at) = o;
  }
}

// W as [64 n][64 k], zeros outside; all threads.
template <typename T>
__device__ __forceinline__ void load_narrow_weights(unsigned char* dst, const NarrowArgs& p) {
  const T* w = static_cast<const T*>(p.w);
  for (int i = threadIdx.x; i < kNarrow * 16; i += kNarrowThreadsL) {
    const int r = i >> 4, u = i & 15;
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      v[j] = r < p.n && 4 * u + j < p.k ? to_float(w[r * p.ldw + 4 * u + j]) : 0.f;
    store_unit<T>(dst, kNarrow * 128, r, u, v);
  }
}

// One slice of a contiguous operand of `width` columns: what of it was copied (whole
// 16-byte blocks) and where the rest is.
template <typename T>
struct Slice {
  const T* raw;     // in shared memory
  const T* global;  // the same elements in memory
  int width, rows;  // rows of the tensor in the slice
  int copied;       // elements

  __device__ __forceinline__ bool whole() const { return copied == rows * width; }
};

template <typename T>
__device__ __forceinline__ uint32_t slice_bytes(int width, int rows) {
  return static_cast<uint32_t>(rows * width * sizeof(T)) & ~15u;
}

// Columns 4 u .. of row r, zeros outside the operand.
template <typename T>
__device__ __forceinline__ void read_unit(const Slice<T>& s, int r, int u, float (&v)[4]) {
  const int at = r * s.width + 4 * u;
  if (r < s.rows && s.whole() && (s.width & 3) == 0) {
    Pack<T, 4> pk{};
    if (4 * u < s.width) pk = *reinterpret_cast<const Pack<T, 4>*>(s.raw + at);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = to_float(pk.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = 0.f;
      if (r < s.rows && 4 * u + j < s.width)
        v[j] = to_float(at + j < s.copied ? s.raw[at + j] : s.global[at + j]);
    }
  }
}

// The `steps` K steps of one product, all the parts' products of a step together; strides
// in the descriptors' units of 16 bytes.
template <int P>
__device__ __forceinline__ void issue_cut(uint32_t d, uint32_t small, uint64_t a, uint64_t a_step,
                                          uint64_t a_part, uint64_t b, uint64_t b_step,
                                          uint64_t b_part, uint32_t desc, int steps, bool add) {
#pragma unroll 1
  for (int k = 0; k < steps; ++k, a += a_step, b += b_step) {
    mma_f16(d, a, b, desc, add);
    if constexpr (P == 3) {
      mma_f16(small, a + 2 * a_part, b, desc, add);
      mma_f16(small, a, b + 2 * b_part, desc, true);
      mma_f16(small, a + a_part, b + b_part, desc, true);
      mma_f16(small, a + a_part, b, desc, true);
      mma_f16(small, a, b + b_part, desc, true);
    }
    add = true;
  }
}

// 32 columns of the warp's TMEM lanes, large and small sums together.
template <int P>
__device__ __forceinline__ void take_sums(uint32_t at, uint32_t small, float (&v)[32], bool add) {
#pragma unroll
  for (int j = 0; j < 32; j += 16) {
    float w[16];
    tmem_load16(at + j, w);
    tmem_load_wait();
#pragma unroll
    for (int i = 0; i < 16; ++i) v[j + i] = add ? v[j + i] + w[i] : w[i];
    if constexpr (P == 3) {
      tmem_load16(at + small + j, w);
      tmem_load_wait();
#pragma unroll
      for (int i = 0; i < 16; ++i) v[j + i] += w[i];
    }
  }
}

__device__ __forceinline__ bool any_nonfinite(const float (&v)[32]) {
  float zero = 0.f;  // stays 0 unless an element is not finite
#pragma unroll
  for (int i = 0; i < 32; ++i) zero = fmaf(v[i], 0.f, zero);
  return zero != 0.f;
}

// The CTA's slices in order, for the thread that issues copies and for those that wait.
struct SliceWalk {
  int tile, slice, tiles, step;
  int64_t m;

  __device__ __forceinline__ bool done() const { return tile >= tiles; }
  __device__ __forceinline__ int64_t row() const {
    return static_cast<int64_t>(tile) * kNarrowTile + slice * kSliceRows;
  }
  __device__ __forceinline__ int rows() const {
    const int64_t left = m - row();
    return left < kSliceRows ? static_cast<int>(left) : kSliceRows;
  }
  __device__ __forceinline__ void next() {
    if (++slice == kNarrowTile / kSliceRows || row() >= m) {
      slice = 0;
      tile += step;
    }
  }
};

// ------------------------------------------------------------------------- forward

// Elements of y that came out NaN or infinite, by FMAs in order (the values are in `mine`).
__device__ __noinline__ void repair_narrow_forward(const NarrowArgs& p, const float* mine,
                                                   int64_t row, int col0, int lane) {
  const float* x = static_cast<const float*>(p.x);
  const float* w = static_cast<const float*>(p.w);
  for (int c = 0; c < 32; ++c) {
    const int col = col0 + c;
    const float v = mine[lane * 32 + (((c >> 2) ^ (lane & 7)) << 2) + (c & 3)];
    if (row >= p.m || col >= p.n || isfinite(v)) continue;
    float s = 0.f;
    for (int k = 0; k < p.k; ++k) s = fmaf(x[row * p.k + k], w[col * p.ldw + k], s);
    finish1<float, kAnyActivation>(p.e, row, col, p.n, s,
                                   p.e.bias ? static_cast<const float*>(p.e.bias)[col] : 0.f);
  }
}

template <typename T, int ACT>
__global__ void __launch_bounds__(kNarrowThreadsL, 1)
    narrow_forward_kernel(const __grid_constant__ NarrowArgs p) {
  constexpr int P = kCut<T>, R = kForwardSlices;
  constexpr uint32_t kSet = (P == 3 ? 2 : 1) * kNarrow, kColumns = 2 * kSet;
  constexpr uint32_t kPiece = kNarrowTile * 128;
  extern __shared__ unsigned char raw_smem[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t{1023});
  unsigned char* weights = smem;
  unsigned char* tiles = weights + kNarrowW<T>;
  unsigned char* slices = tiles + 2 * kNarrowOperand<T>;
  unsigned char* staging = slices + R * kSliceX<T>;
  uint64_t* raw_full = reinterpret_cast<uint64_t*>(staging + kNarrowStaging);
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
      mbar_init(&raw_empty[i], 8);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&full[i], 8);
      mbar_init(&empty[i], 1);
      mbar_init(&done[i], 1);
      mbar_init(&room[i], 8);
    }
    mbar_init(drain, 1);
    fence_mbarrier_init();
  }
  if (warp == 0) tmem_alloc(tmem_at, kColumns);
  load_narrow_weights<T>(weights, p);
  fence_proxy_async();
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = *tmem_at;

  if (warp >= 8) {
    const int tid = threadIdx.x - 256, unit = tid & 15, r0 = tid >> 4;
    const int steps = (p.k + 15) / 16;
    const T* x = static_cast<const T*>(p.x);
    const SliceWalk start{static_cast<int>(blockIdx.x), 0, p.tiles, static_cast<int>(gridDim.x),
                          p.m};
    SliceWalk ahead = start;
    const auto copy = [&](int slot) {  // the next slice to be copied, into `slot`
      if (ahead.done()) return;
      const uint32_t bytes = slice_bytes<T>(p.k, ahead.rows());
      mbar_arrive_expect_tx(&raw_full[slot], bytes);
      if (bytes) bulk_g2s(slices + slot * kSliceX<T>, x + ahead.row() * p.k, bytes,
                          &raw_full[slot]);
      ahead.next();
    };
    const bool copies = warp == kNarrowCopyWarp && lane == 0;
    if (copies)
      for (int i = 0; i < R; ++i) copy(i);
    bool ok = true;
    uint32_t it = 0, n = 0;  // tiles and slices so far
    for (int t = blockIdx.x; ok && t < p.tiles; t += gridDim.x, ++it) {
      const int s = it & 1;
      ok = mbar_wait_warp(&empty[s], ((it >> 1) & 1) ^ 1, kCodeProducer);
      if (!ok) break;
      unsigned char* tile = tiles + s * kNarrowOperand<T>;
      SliceWalk at{t, 0, p.tiles, static_cast<int>(gridDim.x), p.m};
#pragma unroll 1
      for (int q = 0; q < kNarrowTile / kSliceRows; ++q, ++at.slice) {
        Slice<T> slice{nullptr, nullptr, p.k, 0, 0};
        const bool some = at.row() < p.m;
        if (some) {
          const int slot = n % R;
          ok = mbar_wait_warp(&raw_full[slot], (n / R) & 1, kCodeProducer);
          if (!ok) break;
          slice.raw = reinterpret_cast<const T*>(slices + slot * kSliceX<T>);
          slice.global = x + at.row() * p.k;
          slice.rows = at.rows();
          slice.copied = static_cast<int>(slice_bytes<T>(p.k, slice.rows) / sizeof(T));
        }
        float v[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) read_unit(slice, r0 + 16 * j, unit, v[j]);
        if (some) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&raw_empty[n % R]);
        }
        if (unit < 4 * steps)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            store_unit<T>(tile, kPiece, q * kSliceRows + r0 + 16 * j, unit, v[j]);
        if (some) {
          if (copies) {
            ok = mbar_wait(&raw_empty[n % R], (n / R) & 1, kCodeProducer);
            if (ok) copy(n % R);
          }
          if (warp == kNarrowCopyWarp) ok = __shfl_sync(0xffffffffu, static_cast<int>(ok), 0) != 0;
          if (!ok) break;
          ++n;
        }
      }
      if (!ok) break;
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[s]);
      if (warp == kNarrowMmaWarp) {
        if (lane == 0) {
          ok = mbar_wait(&room[s], ((it >> 1) & 1) ^ 1, kCodeMma) &&
               mbar_wait(&full[s], (it >> 1) & 1, kCodeMma);
          if (ok) {
            tcgen05_fence_after();
            constexpr uint32_t kDesc =
                mma_descriptor(!std::is_same_v<T, __half>, false, false, kNarrowTile, kNarrow);
            const uint32_t d = tmem + s * kSet;
            issue_cut<P>(d, d + kNarrow, matrix_descriptor(smem_addr(tile), 0, 1024), 2,
                         kPiece / 16, matrix_descriptor(smem_addr(weights), 0, 1024), 2,
                         kNarrow * 128 / 16, kDesc, steps, false);
            mma_commit(&empty[s]);
            mma_commit(&done[s]);
          }
        }
        ok = __shfl_sync(0xffffffffu, static_cast<int>(ok), 0) != 0;
      }
    }
    if (!ok && (warp == kNarrowMmaWarp || warp == kNarrowCopyWarp)) {
      if (lane == 0 && warp == kNarrowMmaWarp) {  // MMAs in flight finish
        mma_commit(drain);
        mbar_wait(drain, 0, kCodeDrain, kDrainLimitNs);
      } else if (lane == 0) {  // copies in flight land
        const unsigned long long begin = global_timer_ns();
        while (global_timer_ns() - begin < kDrainLimitNs) {
        }
      }
      __syncwarp();
    }
  } else {
    const int quad = warp & 3, half = warp >> 2;
    float4* mine = reinterpret_cast<float4*>(staging + warp * 4096);
    ProductArgs o{};
    o.m = p.m;
    o.n = p.n;
    o.e = p.e;
    uint32_t it = 0;
    for (int t = blockIdx.x; t < p.tiles; t += gridDim.x, ++it) {
      const int s = it & 1;
      const int64_t row0 = static_cast<int64_t>(t) * kNarrowTile + quad * 32;
      ResidualBlock<T> res;
      load_residual(o, row0, half * 32, lane, res);
      if (!mbar_wait_warp(&done[s], (it >> 1) & 1, kCodeEpilogue)) break;
      tcgen05_fence_after();
      float acc[32];
      take_sums<P>(tmem + s * kSet + (static_cast<uint32_t>(quad * 32) << 16) + half * 32, kNarrow,
                   acc, false);
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&room[s]);
      write_block<T, ACT>(o, 0, acc, mine, row0, half * 32, lane, res);
      if constexpr (P == 3) {
        if (__any_sync(0xffffffffu, any_nonfinite(acc)))
          repair_narrow_forward(p, reinterpret_cast<const float*>(mine), row0 + lane, half * 32,
                                lane);
        __syncwarp();
      }
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 0) {
    tcgen05_fence_after();
    tmem_free(tmem, kColumns);
  }
}

// ------------------------------------------------------------------------ backward

template <int ACT>
__device__ __forceinline__ float narrow_d(const NarrowArgs& p, int64_t at) {
  const float g = static_cast<const float*>(p.g)[at];
  return ACT == ICTC_ACT_NONE ? g : g * activation_slope<ACT, false>(p.preact[at]);
}

// As above for dx = d W.
template <int ACT>
__device__ __noinline__ void repair_narrow_dx(const NarrowArgs& p, const float* mine, int64_t row,
                                              int col0, int lane) {
  const float* w = static_cast<const float*>(p.w);
  for (int c = 0; c < 32; ++c) {
    const int col = col0 + c;
    const float v = mine[lane * 32 + (((c >> 2) ^ (lane & 7)) << 2) + (c & 3)];
    if (row >= p.m || col >= p.k || isfinite(v)) continue;
    float s = 0.f;
    for (int n = 0; n < p.n; ++n) s = fmaf(narrow_d<ACT>(p, row * p.n + n), w[n * p.ldw + col], s);
    static_cast<float*>(p.e.out)[row * p.k + col] = s;
  }
}

// One element of the CTA's d^T x, by FMAs over its rows in order.
template <int ACT>
__device__ __noinline__ float repair_narrow_dw(const NarrowArgs& p, int n, int k) {
  const float* x = static_cast<const float*>(p.x);
  float s = 0.f;
  for (int t = blockIdx.x; t < p.tiles; t += gridDim.x)
    for (int r = 0; r < kNarrowTile; ++r) {
      const int64_t row = static_cast<int64_t>(t) * kNarrowTile + r;
      if (row >= p.m) break;
      s = fmaf(narrow_d<ACT>(p, row * p.n + n), x[row * p.k + k], s);
    }
  return s;
}

template <typename T, int ACT>
__global__ void __launch_bounds__(kNarrowThreadsL, 1)
    narrow_backward_kernel(const __grid_constant__ NarrowArgs p) {
  constexpr int P = kCut<T>, R = kBackwardSlices<T>;
  constexpr uint32_t kSet = (P == 3 ? 2 : 1) * kNarrow;
  constexpr uint32_t kColumns = 4 * kSet;  // two sets of dx, two of dW
  constexpr uint32_t kPiece = kNarrowTile * 128;
  extern __shared__ unsigned char raw_smem[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t{1023});
  unsigned char* weights = smem;
  unsigned char* d_tile = weights + kNarrowW<T>;
  unsigned char* x_tile = d_tile + kNarrowOperand<T>;
  unsigned char* slices = x_tile + kNarrowOperand<T>;
  unsigned char* staging = slices + R * kBackwardSlice<T>;
  uint64_t* raw_full = reinterpret_cast<uint64_t*>(staging + kNarrowStaging);
  uint64_t* raw_empty = raw_full + R;
  uint64_t* full = raw_empty + R;
  uint64_t* empty = full + 1;
  uint64_t* done = empty + 1;     // dx sets
  uint64_t* room = done + 2;
  uint64_t* dw_done = room + 2;   // dW sets
  uint64_t* dw_room = dw_done + 2;
  uint64_t* drain = dw_room + 2;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(drain + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < R; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], 8);
    }
    mbar_init(full, 8);
    mbar_init(empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&done[i], 1);
      mbar_init(&room[i], 8);
      mbar_init(&dw_done[i], 1);
      mbar_init(&dw_room[i], 4);
    }
    mbar_init(drain, 1);
    fence_mbarrier_init();
  }
  if (warp == 0) tmem_alloc(tmem_at, kColumns);
  load_narrow_weights<T>(weights, p);
  // columns past n and k are never written again; their products are dropped, but the MMA
  // should not read what was never written
  for (uint32_t i = threadIdx.x; i < 2 * kNarrowOperand<T> / 16; i += kNarrowThreadsL)
    reinterpret_cast<uint4*>(d_tile)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async();
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = *tmem_at;
  const bool want_dx = p.e.out != nullptr, want_dw = p.partial != nullptr;
  float db[4] = {0.f, 0.f, 0.f, 0.f};

  if (warp >= 8) {
    const int tid = threadIdx.x - 256, unit = tid & 15, r0 = tid >> 4;
    const T* x = static_cast<const T*>(p.x);
    const T* g = static_cast<const T*>(p.g);
    SliceWalk ahead{static_cast<int>(blockIdx.x), 0, p.tiles, static_cast<int>(gridDim.x), p.m};
    const auto copy = [&](int slot) {
      if (ahead.done()) return;
      const uint32_t bx = slice_bytes<T>(p.k, ahead.rows());
      const uint32_t bg = slice_bytes<T>(p.n, ahead.rows());
      const uint32_t bp = ACT == ICTC_ACT_NONE ? 0 : slice_bytes<float>(p.n, ahead.rows());
      unsigned char* to = slices + slot * kBackwardSlice<T>;
      mbar_arrive_expect_tx(&raw_full[slot], bx + bg + bp);
      if (bx) bulk_g2s(to, x + ahead.row() * p.k, bx, &raw_full[slot]);
      if (bg) bulk_g2s(to + kSliceX<T>, g + ahead.row() * p.n, bg, &raw_full[slot]);
      if (bp) bulk_g2s(to + 2 * kSliceX<T>, p.preact + ahead.row() * p.n, bp, &raw_full[slot]);
      ahead.next();
    };
    const bool copies = warp == kNarrowCopyWarp && lane == 0;
    if (copies)
      for (int i = 0; i < R; ++i) copy(i);
    bool ok = true;
    uint32_t it = 0, n = 0;
    for (int t = blockIdx.x; ok && t < p.tiles; t += gridDim.x, ++it) {
      // the tile's x and d into registers while the MMAs still read the previous tile
      float xv[8][4], dv[8][4];
      SliceWalk at{t, 0, p.tiles, static_cast<int>(gridDim.x), p.m};
#pragma unroll
      for (int q = 0; q < kNarrowTile / kSliceRows; ++q, ++at.slice) {
        const bool some = ok && at.row() < p.m;
        Slice<T> sx{nullptr, nullptr, p.k, 0, 0}, sg{nullptr, nullptr, p.n, 0, 0};
        Slice<float> sp{nullptr, nullptr, p.n, 0, 0};
        const int slot = n % R;
        if (some) {
          ok = mbar_wait_warp(&raw_full[slot], (n / R) & 1, kCodeProducer);
          const unsigned char* from = slices + slot * kBackwardSlice<T>;
          const int rows = ok ? at.rows() : 0;
          sx = {reinterpret_cast<const T*>(from), x + at.row() * p.k, p.k, rows,
                static_cast<int>(slice_bytes<T>(p.k, rows) / sizeof(T))};
          sg = {reinterpret_cast<const T*>(from + kSliceX<T>), g + at.row() * p.n, p.n, rows,
                static_cast<int>(slice_bytes<T>(p.n, rows) / sizeof(T))};
          sp = {reinterpret_cast<const float*>(from + 2 * kSliceX<T>), p.preact + at.row() * p.n,
                p.n, rows, static_cast<int>(slice_bytes<float>(p.n, rows) / sizeof(float))};
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          read_unit(sx, r0 + 16 * j, unit, xv[2 * q + j]);
          float(&d)[4] = dv[2 * q + j];
          read_unit(sg, r0 + 16 * j, unit, d);
          if constexpr (ACT != ICTC_ACT_NONE) {
            float pv[4];
            read_unit(sp, r0 + 16 * j, unit, pv);
#pragma unroll
            for (int i = 0; i < 4; ++i) d[i] *= activation_slope<ACT, sizeof(T) == 2>(pv[i]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) db[i] += d[i];
        }
        if (some) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&raw_empty[slot]);
          if (copies && ok) {
            ok = mbar_wait(&raw_empty[slot], (n / R) & 1, kCodeProducer);
            if (ok) copy(slot);
          }
          if (warp == kNarrowCopyWarp) ok = __shfl_sync(0xffffffffu, static_cast<int>(ok), 0) != 0;
          ++n;
        }
      }
      if (ok) ok = mbar_wait_warp(empty, (it & 1) ^ 1, kCodeProducer);
      if (!ok) break;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = (i >> 1) * kSliceRows + r0 + 16 * (i & 1);
        if (4 * unit < p.k) store_unit<T>(x_tile, kPiece, r, unit, xv[i]);
        if (4 * unit < p.n) store_unit<T>(d_tile, kPiece, r, unit, dv[i]);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(full);
      if (warp == kNarrowMmaWarp) {
        if (lane == 0) {
          constexpr bool kBf16 = !std::is_same_v<T, __half>;
          const uint32_t da = smem_addr(d_tile), xa = smem_addr(x_tile), wa = smem_addr(weights);
          ok = mbar_wait(full, it & 1, kCodeMma);
          if (ok && want_dx) {
            const int s = it & 1;
            ok = mbar_wait(&room[s], ((it >> 1) & 1) ^ 1, kCodeMma);
            if (ok) {
              tcgen05_fence_after();
              // W as [n][k] is MN-major for the sum over n: 16 rows a step
              constexpr uint32_t kDesc = mma_descriptor(kBf16, false, true, kNarrowTile, kNarrow);
              const uint32_t acc = tmem + s * kSet;
              issue_cut<P>(acc, acc + kNarrow, matrix_descriptor(da, 0, 1024), 2, kPiece / 16,
                           matrix_descriptor(wa, 0, 1024), 128, kNarrow * 128 / 16, kDesc,
                           (p.n + 15) / 16, false);
              mma_commit(&done[s]);
            }
          }
          if (ok && want_dw) {
            const uint32_t group = it / kDwTiles, s = group & 1;
            const bool first = it % kDwTiles == 0;
            if (first) ok = mbar_wait(&dw_room[s], ((group >> 1) & 1) ^ 1, kCodeMma);
            if (ok) {
              tcgen05_fence_after();
              // both operands MN-major over the tile's rows; M is d's 64 columns and, one
              // operand further, x's
              constexpr uint32_t kDesc = mma_descriptor(kBf16, true, true, 128, kNarrow);
              const uint32_t acc = tmem + 2 * kSet + s * kSet;
              issue_cut<P>(acc, acc + kNarrow, matrix_descriptor(da, kNarrowOperand<T>, 1024), 128,
                           kPiece / 16, matrix_descriptor(xa, 0, 1024), 128, kPiece / 16, kDesc,
                           kNarrowTile / 16, !first);
              if (it % kDwTiles == kDwTiles - 1 ||
                  t + static_cast<int>(gridDim.x) >= p.tiles)
                mma_commit(&dw_done[s]);
            }
          }
          if (ok) mma_commit(empty);
        }
        ok = __shfl_sync(0xffffffffu, static_cast<int>(ok), 0) != 0;
      }
    }
    if (!ok && (warp == kNarrowMmaWarp || warp == kNarrowCopyWarp)) {
      if (lane == 0 && warp == kNarrowMmaWarp) {
        mma_commit(drain);
        mbar_wait(drain, 0, kCodeDrain, kDrainLimitNs);
      } else if (lane == 0) {
        const unsigned long long begin = global_timer_ns();
        while (global_timer_ns() - begin < kDrainLimitNs) {
        }
      }
      __syncwarp();
    }
  } else {
    const int quad = warp & 3, half = warp >> 2;
    float4* mine = reinterpret_cast<float4*>(staging + warp * 4096);
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    ProductArgs o{};
    o.m = p.m;
    o.n = p.k;
    o.e = p.e;
    const ResidualBlock<T> none{};
    float dw[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) dw[i] = 0.f;
    bool ok = true;
    uint32_t it = 0;
    for (int t = blockIdx.x; ok && t < p.tiles; t += gridDim.x, ++it) {
      if (want_dx) {
        const int s = it & 1;
        const int64_t row0 = static_cast<int64_t>(t) * kNarrowTile + quad * 32;
        ok = mbar_wait_warp(&done[s], (it >> 1) & 1, kCodeEpilogue);
        if (!ok) break;
        tcgen05_fence_after();
        float acc[32];
        take_sums<P>(tmem + s * kSet + lanes + half * 32, kNarrow, acc, false);
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&room[s]);
        write_block<T, ICTC_ACT_NONE>(o, 0, acc, mine, row0, half * 32, lane, none);
        if constexpr (P == 3) {
          if (__any_sync(0xffffffffu, any_nonfinite(acc)))
            repair_narrow_dx<ACT>(p, reinterpret_cast<const float*>(mine), row0 + lane, half * 32,
                                  lane);
          __syncwarp();
        }
      }
      if (want_dw && quad < 2 &&
          (it % kDwTiles == kDwTiles - 1 || t + static_cast<int>(gridDim.x) >= p.tiles)) {
        const uint32_t group = it / kDwTiles, s = group & 1;
        ok = mbar_wait_warp(&dw_done[s], (group >> 1) & 1, kCodeEpilogue);
        if (!ok) break;
        tcgen05_fence_after();
        take_sums<P>(tmem + 2 * kSet + s * kSet + lanes + half * 32, kNarrow, dw, true);
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&dw_room[s]);
      }
    }
    if (want_dw && quad < 2) {
      const int n = quad * 32 + lane;
      float* out = p.partial + static_cast<int64_t>(blockIdx.x) * (p.n * p.k + p.n);
      if (n < p.n)
        for (int i = 0; i < 32; ++i) {
          const int k = half * 32 + i;
          float v = 0.f;
#pragma unroll
          for (int j = 0; j < 32; ++j) v = i == j ? dw[j] : v;
          if (k >= p.k) break;
          if constexpr (P == 3) {
            if (!isfinite(v)) v = repair_narrow_dw<ACT>(p, n, k);
          }
          out[n * p.k + k] = v;
        }
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 0) {
    tcgen05_fence_after();
    tmem_free(tmem, kColumns);
  }
  // db: the 16 row lanes of each column, in order (the slices are free now)
  if (!want_dw) return;
  float* sums = reinterpret_cast<float*>(slices);
  if (warp >= 8) {
    const int tid = threadIdx.x - 256;
    *reinterpret_cast<float4*>(sums + (tid >> 4) * kNarrow + (tid & 15) * 4) =
        make_float4(db[0], db[1], db[2], db[3]);
  }
  __syncthreads();
  if (threadIdx.x < p.n) {
    float total = 0.f;
    for (int q = 0; q < 16; ++q) total += sums[q * kNarrow + threadIdx.x];
    p.partial[static_cast<int64_t>(blockIdx.x) * (p.n * p.k + p.n) + p.n * p.k + threadIdx.x] =
        total;
  }
}

// dW and db from the CTAs' partial rows [parts][nk + n]; lanes and order as
// column_total_kernel.
template <typename T>
static __global__ void __launch_bounds__(32 * kColumnLanes)
    narrow_total_kernel(const float* __restrict__ partial, T* __restrict__ dw, T* __restrict__ db,
                        int parts, int nk, int n) {
  __shared__ float sums[kColumnLanes][33];
  const int c = blockIdx.x * 32 + threadIdx.x, width = nk + n;
  float s = 0.f;
  if (c < width)
#pragma unroll 4
    for (int p = threadIdx.y; p < parts; p += kColumnLanes)
      s += partial[static_cast<int64_t>(p) * width + c];
  sums[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < width) {
    float total = 0.f;
    for (int l = 0; l < kColumnLanes; ++l) total += sums[l][threadIdx.x];
    if (c < nk) {
      if (dw) dw[c] = from_float<T>(total);
    } else if (db) {
      db[c - nk] = from_float<T>(total);
    }
  }
}

}  // namespace ictc
