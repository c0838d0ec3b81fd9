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
//
// float32, 1,048,576 x 64 x 64 with SiLU and residual: forward 194 us (x, r, y, p: 1.07 GB,
// 5.5 TB/s), backward 270 us (x, g, p, dx: 1.07 GB, 4.0 TB/s), where the cutting of x and d by
// the producer warps is what is left over HBM.
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

// Warps of a CTA: epilogue first, then producers, one that issues the MMAs and one that
// starts the copies.  Fourteen of them leave a thread 128 registers.  (The MMA queue
// holds its issuer back while it is full: with a producer as the issuer the next tile's
// slices waited for it, and the float32 backward of 1,048,576 rows took 584 instead of
// 337 us.)
constexpr int kNarrowWarps = 14;
constexpr int kNarrowThreadsL = kNarrowWarps * 32;
constexpr int kNarrowMmaWarp = 12, kNarrowCopyWarp = 13;
constexpr int kForwardEpilogue = 8, kBackwardEpilogue = 4;
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
constexpr uint32_t kNarrowStaging = 8 * 4096;  // 4 KB per epilogue warp, at most eight

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
    uint32_t lo[3], hi[3];
    cut_pair(v[0], v[1], lo);
    cut_pair(v[2], v[3], hi);
#pragma unroll
    for (int q = 0; q < 3; ++q)
      *reinterpret_cast<uint2*>(at + q * piece) = make_uint2(lo[q], hi[q]);
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
};

template <typename T>
__device__ __forceinline__ uint32_t slice_bytes(int width, int rows) {
  return static_cast<uint32_t>(rows * width * sizeof(T)) & ~15u;
}

template <typename T>
__device__ __noinline__ float4 read_unit_edge(const T* raw, const T* global, int width, int rows,
                                              int copied, int r, int u) {
  float v[4];
  const int at = r * width + 4 * u;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[j] = 0.f;
    if (r < rows && 4 * u + j < width)
      v[j] = to_float(at + j < copied ? raw[at + j] : global[at + j]);
  }
  return make_float4(v[0], v[1], v[2], v[3]);
}

// One value out of shared memory.
template <typename T>
__device__ __forceinline__ float read_shared(uint32_t at) {
  if constexpr (sizeof(T) == 4) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
  } else {
    uint16_t bits;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(bits) : "r"(at) : "memory");
    return to_float(*reinterpret_cast<const T*>(&bits));
  }
}

// Columns 4 u .. of row r, zeros outside the operand.  PLAIN: rows are whole 16-byte
// blocks, and a unit is one access; a kernel of its own, because the general read's code
// between the others' cost a third of the time.  Otherwise its values are read one by one;
// 32 rows of any width are whole blocks, so only a tensor's last slice can have values that
// were not copied.
template <bool PLAIN, typename T>
__device__ __forceinline__ void read_unit(const Slice<T>& s, int r, int u, float (&v)[4]) {
  if constexpr (PLAIN) {
    uint32_t q[4] = {0, 0, 0, 0};
    if (r < s.rows && 4 * u < s.width) {
      const uint32_t at = smem_addr(s.raw) + (r * s.width + 4 * u) * sizeof(T);
      if constexpr (sizeof(T) == 4)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3])
                     : "r"(at)
                     : "memory");
      else
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];"
                     : "=r"(q[0]), "=r"(q[1])
                     : "r"(at)
                     : "memory");
    }
    const Pack<T, 4>& pk = *reinterpret_cast<const Pack<T, 4>*>(q);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = to_float(pk.v[j]);
  } else if (s.copied == s.rows * s.width) {
    const uint32_t at = smem_addr(s.raw) + (r * s.width + 4 * u) * sizeof(T);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = 0.f;
      if (r < s.rows && 4 * u + j < s.width) v[j] = read_shared<T>(at + j * sizeof(T));
    }
  } else {
    const float4 f = read_unit_edge(s.raw, s.global, s.width, s.rows, s.copied, r, u);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  }
}

// Bits of every value of a unit, for release_slot: a PLAIN unit is one access, whose first
// value arrives with the other three; elsewhere each value has a load of its own.
template <bool PLAIN>
__device__ __forceinline__ uint32_t unit_bits(const float (&v)[4]) {
  const uint32_t first = __float_as_uint(v[0]);
  if constexpr (PLAIN) return first;
  return first | __float_as_uint(v[1]) | __float_as_uint(v[2]) | __float_as_uint(v[3]);
}

// The `steps` K steps of one product with 64 columns; strides in the descriptors' units of
// 16 bytes.  The parts of B lie behind one another as 192 columns, so that a part of A
// meets all the parts of B that it needs in one MMA, which fetches A again every time:
//   a1 (b1 | b2 | b3), a2 (b1 | b2), a3 b1   into sums of order 0, 1 and 2, 64 columns each.
template <int P>
__device__ __forceinline__ void issue_cut(uint32_t d, uint64_t a, uint64_t a_step, uint64_t a_part,
                                          uint64_t b, uint64_t b_step, bool bf16, bool a_mn,
                                          bool b_mn, int steps, bool add) {
  const uint32_t one = mma_descriptor(bf16, a_mn, b_mn, kNarrowTile, kNarrow);
  const uint32_t two = mma_descriptor(bf16, a_mn, b_mn, kNarrowTile, 2 * kNarrow);
  const uint32_t three = mma_descriptor(bf16, a_mn, b_mn, kNarrowTile, 3 * kNarrow);
#pragma unroll 1
  for (int k = 0; k < steps; ++k, a += a_step, b += b_step) {
    if constexpr (P == 3) {
      mma_f16(d, a, b, three, add);
      mma_f16(d + kNarrow, a + a_part, b, two, true);
      mma_f16(d + 2 * kNarrow, a + 2 * a_part, b, one, true);
    } else {
      mma_f16(d, a, b, one, add);
    }
    add = true;
  }
}

// 32 columns of the warp's TMEM lanes, the sums of all orders together.
template <int P>
__device__ __forceinline__ void take_sums(uint32_t at, float (&v)[32], bool add) {
#pragma unroll
  for (int j = 0; j < 32; j += 16) {
    float w[16], y[16];
    if constexpr (P == 3) {
      tmem_load16(at + kNarrow + j, y);
      tmem_load16(at + 2 * kNarrow + j, w);
      tmem_load_wait();
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] += w[i];
    }
    tmem_load16(at + j, w);
    tmem_load_wait();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float sum = P == 3 ? join_parts(w[i], y[i]) : w[i];
      v[j + i] = add ? v[j + i] + sum : sum;
    }
  }
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

// A producer warp is done with a slot.  `seen` holds bits of every load that the lane made
// from it (unit_bits), and the arrival depends on it: the assembler had moved reads whose values were
// used later behind a plain arrival, where the next copy overwrote the slot first (one row
// in some hundred thousand of the forward was another slice's).  The pattern is that of no
// finite value, and lanes agree on it only if all 32 hold it.
__device__ __forceinline__ void release_slot(uint64_t* bar, uint32_t seen, int lane) {
  const uint32_t alike = __ballot_sync(0xffffffffu, seen == 0xffedcba9u);
  if (lane == (alike == 0xffffffffu ? 1 : 0)) mbar_arrive(bar);
}

// Copies in flight land before the CTA goes away (after a wait ran out).
__device__ __forceinline__ void settle_copies() {
  const unsigned long long begin = global_timer_ns();
  while (global_timer_ns() - begin < kDrainLimitNs) {
  }
}

// ------------------------------------------------------------------------- forward

template <typename T, int ACT, bool PLAIN>
__global__ void __launch_bounds__(kNarrowThreadsL, 1)
    narrow_forward_kernel(const __grid_constant__ NarrowArgs p) {
  constexpr int P = kCut<T>, R = kForwardSlices;
  constexpr uint32_t kSet = P * kNarrow, kColumns = P == 3 ? 512 : 2 * kSet;
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
    constexpr int kProducers = kNarrowMmaWarp - kForwardEpilogue;
    for (int i = 0; i < R; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], kProducers);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&full[i], kProducers);
      mbar_init(&empty[i], 1);
      mbar_init(&done[i], 1);
      mbar_init(&room[i], kForwardEpilogue);
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

  const int steps = (p.k + 15) / 16;
  if (warp == kNarrowCopyWarp) {
    if (lane == 0) {
      const T* x = static_cast<const T*>(p.x);
      SliceWalk at{static_cast<int>(blockIdx.x), 0, p.tiles, static_cast<int>(gridDim.x), p.m};
      bool ok = true;
      for (uint32_t n = 0; !at.done(); at.next(), ++n) {
        const int slot = n % R;
        ok = mbar_wait_idle(&raw_empty[slot], ((n / R) & 1) ^ 1, kCodeProducer);
        if (!ok) break;
        const uint32_t bytes = slice_bytes<T>(p.k, at.rows());
        mbar_arrive_expect_tx(&raw_full[slot], bytes);
        if (bytes)
          bulk_g2s(slices + slot * kSliceX<T>, x + at.row() * p.k, bytes, &raw_full[slot]);
      }
      if (!ok) settle_copies();
    }
    __syncwarp();
  } else if (warp == kNarrowMmaWarp) {
    if (lane == 0) {
      bool ok = true;
      uint32_t it = 0;
      for (int t = blockIdx.x; t < p.tiles; t += gridDim.x, ++it) {
        const int s = it & 1;
        ok = mbar_wait_idle(&room[s], ((it >> 1) & 1) ^ 1, kCodeMma) &&
             mbar_wait_idle(&full[s], (it >> 1) & 1, kCodeMma);
        if (!ok) break;
        tcgen05_fence_after();
        issue_cut<P>(tmem + s * kSet,
                     matrix_descriptor(smem_addr(tiles + s * kNarrowOperand<T>), 0, 1024), 2,
                     kPiece / 16, matrix_descriptor(smem_addr(weights), 0, 1024), 2,
                     !std::is_same_v<T, __half>, false, false, steps, false);
        mma_commit(&empty[s]);
        mma_commit(&done[s]);
      }
      if (!ok) {  // MMAs in flight finish
        mma_commit(drain);
        mbar_wait(drain, 0, kCodeDrain, kDrainLimitNs);
      }
    }
    __syncwarp();
  } else if (warp >= kForwardEpilogue) {
    const int tid = threadIdx.x - kForwardEpilogue * 32, unit = tid & 15, r0 = tid >> 4;
    const T* x = static_cast<const T*>(p.x);
    uint32_t it = 0, n = 0;  // tiles and slices so far
    bool ok = true;
    for (int t = blockIdx.x; ok && t < p.tiles; t += gridDim.x, ++it) {
      const int s = it & 1;
      ok = mbar_wait_warp(&empty[s], ((it >> 1) & 1) ^ 1, kCodeProducer);
      unsigned char* tile = tiles + s * kNarrowOperand<T>;
      SliceWalk at{t, 0, p.tiles, static_cast<int>(gridDim.x), p.m};
#pragma unroll 1
      for (int q = 0; ok && q < kNarrowTile / kSliceRows; ++q, ++at.slice) {
        Slice<T> slice{nullptr, nullptr, p.k, 0, 0};
        const bool some = at.row() < p.m;
        const int slot = n % R;
        if (some) {
          ok = mbar_wait_warp(&raw_full[slot], (n / R) & 1, kCodeProducer);
          if (!ok) break;
          slice.raw = reinterpret_cast<const T*>(slices + slot * kSliceX<T>);
          slice.global = x + at.row() * p.k;
          slice.rows = at.rows();
          slice.copied = static_cast<int>(slice_bytes<T>(p.k, slice.rows) / sizeof(T));
        }
        float v[4][4];
        uint32_t seen = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          read_unit<PLAIN>(slice, r0 + 8 * j, unit, v[j]);
          seen |= unit_bits<PLAIN>(v[j]);
        }
        if (unit < 4 * steps)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            store_unit<T>(tile, kPiece, q * kSliceRows + r0 + 8 * j, unit, v[j]);
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
  } else {
    const int quad = warp & 3, half = warp >> 2;
    float4* mine = reinterpret_cast<float4*>(staging + warp * 4096);
    ProductArgs o{};
    o.m = p.m;
    o.n = p.n;
    o.e = p.e;
    uint32_t it = 0;
    // a tile's residual is loaded as soon as the tile before it is written, ahead of the wait
    // for its products (earlier still, the registers of two residuals spill: 225 us)
    ResidualBlock<T> res;
    load_residual(o, static_cast<int64_t>(blockIdx.x) * kNarrowTile + quad * 32, half * 32, lane,
                  res);
    for (int t = blockIdx.x; t < p.tiles; t += gridDim.x, ++it) {
      const int s = it & 1;
      const int64_t row0 = static_cast<int64_t>(t) * kNarrowTile + quad * 32;
      if (!mbar_wait_warp(&done[s], (it >> 1) & 1, kCodeEpilogue)) break;
      tcgen05_fence_after();
      float acc[32];
      take_sums<P>(tmem + s * kSet + (static_cast<uint32_t>(quad * 32) << 16) + half * 32, acc,
                   false);
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&room[s]);
      stage_block(acc, mine, lane);
      write_staged<T, ACT>(o, 0, mine, row0, half * 32, lane, res);
      load_residual(o, row0 + static_cast<int64_t>(gridDim.x) * kNarrowTile, half * 32, lane, res);
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

template <typename T, int ACT, bool PLAIN>
__global__ void __launch_bounds__(kNarrowThreadsL, 1)
    narrow_backward_kernel(const __grid_constant__ NarrowArgs p) {
  constexpr int P = kCut<T>, R = kBackwardSlices<T>;
  constexpr uint32_t kSet = P * kNarrow;
  constexpr uint32_t kColumns = P == 3 ? 512 : 2 * kSet;  // one set of dx, one of dW
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
  uint64_t* x_empty = full + 1;   // x's tile may be written again,
  uint64_t* d_empty = x_empty + 1;  // and d's
  uint64_t* done = d_empty + 1;   // dx
  uint64_t* room = done + 1;
  uint64_t* dw_done = room + 1;   // dW
  uint64_t* dw_room = dw_done + 1;
  uint64_t* drain = dw_room + 1;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(drain + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    constexpr int kProducers = kNarrowMmaWarp - kBackwardEpilogue;
    for (int i = 0; i < R; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], kProducers);
    }
    mbar_init(full, kProducers);
    mbar_init(x_empty, 1);
    mbar_init(d_empty, 1);
    mbar_init(done, 1);
    mbar_init(room, kBackwardEpilogue);
    mbar_init(dw_done, 1);
    mbar_init(dw_room, 2);  // the warps of lanes 0-63
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

  const T* x = static_cast<const T*>(p.x);
  const T* g = static_cast<const T*>(p.g);
  if (warp == kNarrowCopyWarp) {
    if (lane == 0) {
      SliceWalk at{static_cast<int>(blockIdx.x), 0, p.tiles, static_cast<int>(gridDim.x), p.m};
      bool ok = true;
      for (uint32_t n = 0; !at.done(); at.next(), ++n) {
        const int slot = n % R;
        ok = mbar_wait_idle(&raw_empty[slot], ((n / R) & 1) ^ 1, kCodeProducer);
        if (!ok) break;
        const uint32_t bx = slice_bytes<T>(p.k, at.rows());
        const uint32_t bg = slice_bytes<T>(p.n, at.rows());
        const uint32_t bp = ACT == ICTC_ACT_NONE ? 0 : slice_bytes<float>(p.n, at.rows());
        unsigned char* to = slices + slot * kBackwardSlice<T>;
        mbar_arrive_expect_tx(&raw_full[slot], bx + bg + bp);
        if (bx) bulk_g2s(to, x + at.row() * p.k, bx, &raw_full[slot]);
        if (bg) bulk_g2s(to + kSliceX<T>, g + at.row() * p.n, bg, &raw_full[slot]);
        if (bp) bulk_g2s(to + 2 * kSliceX<T>, p.preact + at.row() * p.n, bp, &raw_full[slot]);
      }
      if (!ok) settle_copies();
    }
    __syncwarp();
  } else if (warp == kNarrowMmaWarp) {
    if (lane == 0) {
      constexpr bool kBf16 = !std::is_same_v<T, __half>;
      const uint32_t da = smem_addr(d_tile), xa = smem_addr(x_tile), wa = smem_addr(weights);
      bool ok = true;
      uint32_t it = 0;
      for (int t = blockIdx.x; t < p.tiles; t += gridDim.x, ++it) {
        ok = mbar_wait_idle(full, it & 1, kCodeMma);
        if (!ok) break;
        // dW first: x's tile is free again while the MMAs of dx still read d's
        if (want_dw) {
          const uint32_t group = it / kDwTiles;
          const bool first = it % kDwTiles == 0;
          if (first) ok = mbar_wait_idle(dw_room, (group & 1) ^ 1, kCodeMma);
          if (!ok) break;
          tcgen05_fence_after();
          // both operands MN-major over the tile's rows; M is d's 64 columns and, one
          // operand further, x's; N is x's columns, one part of x after the other
          issue_cut<P>(tmem + kSet, matrix_descriptor(da, kNarrowOperand<T>, 1024), 128,
                       kPiece / 16, matrix_descriptor(xa, kPiece, 1024), 128, kBf16, true, true,
                       kNarrowTile / 16, !first);
          if (it % kDwTiles == kDwTiles - 1 || t + static_cast<int>(gridDim.x) >= p.tiles)
            mma_commit(dw_done);
        }
        mma_commit(x_empty);
        if (want_dx) {
          ok = mbar_wait_idle(room, (it & 1) ^ 1, kCodeMma);
          if (!ok) break;
          tcgen05_fence_after();
          // W as [n][k] is MN-major for the sum over n: 16 rows a step
          issue_cut<P>(tmem, matrix_descriptor(da, 0, 1024), 2, kPiece / 16,
                       matrix_descriptor(wa, kNarrow * 128, 1024), 128, kBf16, false, true,
                       (p.n + 15) / 16, false);
          mma_commit(done);
        }
        mma_commit(d_empty);
      }
      if (!ok) {  // MMAs in flight finish
        mma_commit(drain);
        mbar_wait(drain, 0, kCodeDrain, kDrainLimitNs);
      }
    }
    __syncwarp();
  } else if (warp >= kBackwardEpilogue) {
    const int tid = threadIdx.x - kBackwardEpilogue * 32, unit = tid & 15, r0 = tid >> 4;
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
        uint32_t seen = 0;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          read_unit<PLAIN>(sx, r0 + 16 * j, unit, xv[2 * q + j]);
          float(&d)[4] = dv[2 * q + j];
          read_unit<PLAIN>(sg, r0 + 16 * j, unit, d);
          if constexpr (ACT != ICTC_ACT_NONE) {
            float pv[4];
            read_unit<PLAIN>(sp, r0 + 16 * j, unit, pv);
#pragma unroll
            for (int i = 0; i < 4; ++i) d[i] *= activation_slope<ACT>(pv[i]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) db[i] += d[i];
          seen |= unit_bits<PLAIN>(xv[2 * q + j]) | unit_bits<PLAIN>(d);  // d from g and p
        }
        if (some) {
          release_slot(&raw_empty[slot], seen, lane);
          ++n;
        }
      }
      if (ok) ok = mbar_wait_warp(x_empty, (it & 1) ^ 1, kCodeProducer);
      if (!ok) break;
      const auto row = [&](int i) { return (i >> 1) * kSliceRows + r0 + 16 * (i & 1); };
      if (4 * unit < p.k)
#pragma unroll
        for (int i = 0; i < 8; ++i) store_unit<T>(x_tile, kPiece, row(i), unit, xv[i]);
      ok = mbar_wait_warp(d_empty, (it & 1) ^ 1, kCodeProducer);
      if (!ok) break;
      if (4 * unit < p.n)
#pragma unroll
        for (int i = 0; i < 8; ++i) store_unit<T>(d_tile, kPiece, row(i), unit, dv[i]);
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(full);
    }
  } else {
    const int quad = warp;
    float4* mine = reinterpret_cast<float4*>(staging + warp * 4096);
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    ProductArgs o{};
    o.m = p.m;
    o.n = p.k;
    o.e = p.e;
    const ResidualBlock<T> none{};
    float dw[2][32];
#pragma unroll
    for (int i = 0; i < 32; ++i) dw[0][i] = dw[1][i] = 0.f;
    bool ok = true;
    uint32_t it = 0;
    for (int t = blockIdx.x; ok && t < p.tiles; t += gridDim.x, ++it) {
      if (want_dw && quad < 2 &&
          (it % kDwTiles == kDwTiles - 1 || t + static_cast<int>(gridDim.x) >= p.tiles)) {
        ok = mbar_wait_warp(dw_done, (it / kDwTiles) & 1, kCodeEpilogue);
        if (!ok) break;
        tcgen05_fence_after();
        take_sums<P>(tmem + kSet + lanes, dw[0], true);
        take_sums<P>(tmem + kSet + lanes + 32, dw[1], true);
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(dw_room);
      }
      if (want_dx) {
        const int64_t row0 = static_cast<int64_t>(t) * kNarrowTile + quad * 32;
        ok = mbar_wait_warp(done, it & 1, kCodeEpilogue);
        if (!ok) break;
        tcgen05_fence_after();
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          float acc[32];
          take_sums<P>(tmem + lanes + half * 32, acc, false);
          if (half == 1) {
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(room);
          }
          if (half * 32 >= p.k) continue;
          stage_block(acc, mine, lane);
          write_staged<T, ICTC_ACT_NONE>(o, 0, mine, row0, half * 32, lane, none);
        }
      }
    }
    if (want_dw && quad < 2) {
      const int n = quad * 32 + lane;
      float* out = p.partial + static_cast<int64_t>(blockIdx.x) * (p.n * p.k + p.n);
      if (n < p.n)
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const int k = half * 32 + i;
            if (k < p.k) out[n * p.k + k] = dw[half][i];
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
  if (warp >= kBackwardEpilogue && warp < kNarrowMmaWarp) {
    const int tid = threadIdx.x - kBackwardEpilogue * 32;
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
