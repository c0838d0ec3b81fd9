// Tile order and epilogue shared by the kernels of the linear layer's products.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "dense_types.cuh"

namespace ictc {

// Bounded-wait codes of the products.
constexpr int kCodeProducer = 18, kCodeMma = 19, kCodeEpilogue = 20, kCodeDrain = 21;

struct Epilogue {
  const void* bias;      // [n] or null
  const void* residual;  // [m, n] or null
  int64_t residual_stride;
  float* preact;         // [m, n] p, or null
  void* out;             // [m, n]
  float* partial;        // [splits][m][n] instead of out when the K axis is split
  int activation;
  bool vec;              // four columns per access
};

// C[m, n] = sum over k of A(m, k) B(n, k)
struct ProductArgs {
  const void *a, *b;
  int64_t m, n, k;
  int64_t lda, ldb;      // distance of rows (K-major) or of k (MN-major), in elements
  int tiles_m, tiles_n, splits, chunks, chunks_per_split;
  bool vec_a, vec_b;     // every 8-element chunk inside the operand is 16-byte aligned
  Epilogue e;
};

struct TilePos {
  int64_t m0, n0;
  int split, c0, c1;
};

// Work item t: the splits of K outermost; tiles in bands of eight row tiles, so that the
// CTAs that run together share rows of A and of B in L2.
template <int BM>
__device__ __forceinline__ TilePos tile_at(const ProductArgs& p, int64_t t, int bn) {
  const int64_t tiles = static_cast<int64_t>(p.tiles_m) * p.tiles_n;
  TilePos pos;
  pos.split = static_cast<int>(t / tiles);
  const int64_t r = t - pos.split * tiles;
  const int64_t band = r / (8ll * p.tiles_n);
  const int64_t first = band * 8;
  const int64_t high = p.tiles_m - first < 8 ? p.tiles_m - first : 8;
  const int64_t q = r - band * 8 * p.tiles_n;
  pos.m0 = (first + q % high) * BM;
  pos.n0 = (q / high) * bn;
  pos.c0 = pos.split * p.chunks_per_split;
  pos.c1 = pos.c0 + p.chunks_per_split < p.chunks ? pos.c0 + p.chunks_per_split : p.chunks;
  return pos;
}


// The residual's four columns of a row (vec epilogues).
template <typename T>
__device__ __forceinline__ Pack<T, 4> residual4(const Epilogue& e, int64_t row, int64_t col) {
  return *reinterpret_cast<const Pack<T, 4>*>(static_cast<const T*>(e.residual) +
                                              row * e.residual_stride + col);
}

template <typename T>
__device__ __forceinline__ void load_bias4(const Epilogue& e, int64_t col, int64_t n,
                                           float (&bias)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    bias[j] = e.bias && col + j < n ? to_float(static_cast<const T*>(e.bias)[col + j]) : 0.f;
}

// One column of a row: bias, p, activation, residual and the store of y.
template <typename T, int ACT>
__device__ __forceinline__ void finish1(const Epilogue& e, int64_t row, int64_t col, int64_t n,
                                        float v, float bias) {
  v += bias;
  if (e.preact) e.preact[row * n + col] = v;
  float y = activate<ACT>(v, e.activation);
  if (e.residual) y += to_float(static_cast<const T*>(e.residual)[row * e.residual_stride + col]);
  static_cast<T*>(e.out)[row * n + col] = from_float<T>(y);
}

// Four columns of a row with 16-byte (float32) or 8-byte accesses; r is the residual's, 0
// without one.
template <typename T, int ACT>
__device__ __forceinline__ void finish4(const Epilogue& e, int64_t at, float (&v)[4],
                                        const float (&bias)[4], const Pack<T, 4>& r) {
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] += bias[j];
  if (e.preact) *reinterpret_cast<float4*>(e.preact + at) = make_float4(v[0], v[1], v[2], v[3]);
  Pack<T, 4> o;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    o.v[j] = from_float<T>(activate<ACT>(v[j], e.activation) + to_float(r.v[j]));
  *reinterpret_cast<Pack<T, 4>*>(static_cast<T*>(e.out) + at) = o;
}

// The residual's part of a 32 x 32 block: with a vec epilogue rows lane / 8 + 4 i, four
// columns each; otherwise column `lane`, element j of v[i] row 4 i + j.  Loaded well before
// write_staged needs it (ahead of the wait for the accumulators): loads behind the stores,
// which they might alias, had exposed their latency row by row.
template <typename T>
struct ResidualBlock {
  Pack<T, 4> v[8];
};

template <typename T, int COUNT>
__device__ __forceinline__ void load_residual_part(const ProductArgs& p, int64_t row0,
                                                   int64_t col0, int lane, int first,
                                                   Pack<T, 4>* v) {
  const Epilogue& e = p.e;
  if (!e.residual || e.partial) return;
  const int64_t col = col0 + (e.vec ? (lane & 7) * 4 : lane);
  if (col >= p.n) return;
  const T* base = static_cast<const T*>(e.residual) + col;
  if (e.vec) {
    const int64_t row = row0 + (lane >> 3) + 4 * first;
    const T* at = base + row * e.residual_stride;
#pragma unroll
    for (int i = 0; i < COUNT; ++i)
      if (row + 4 * i < p.m)
        v[i] = *reinterpret_cast<const Pack<T, 4>*>(at + 4 * i * e.residual_stride);
  } else {
    const int64_t row = row0 + 4 * first;
    const T* at = base + row * e.residual_stride;
#pragma unroll
    for (int i = 0; i < 4 * COUNT; ++i)
      if (row + i < p.m) v[i / 4].v[i % 4] = at[i * e.residual_stride];
  }
}

template <typename T>
__device__ __forceinline__ void load_residual(const ProductArgs& p, int64_t row0, int64_t col0,
                                              int lane, ResidualBlock<T>& res) {
  load_residual_part<T, 8>(p, row0, col0, lane, 0, res.v);
}

// One 32 x 32 block of an output tile, row-per-lane in `acc`, to memory: through the
// warp's 4 KB of shared memory (16-byte chunks XOR-swizzled by row), so that lanes of
// one row touch consecutive columns: eight lanes four columns each when the rows are
// aligned for that, 32 lanes one column each otherwise.
__device__ __forceinline__ void stage_block(const float* acc, float4* mine, int lane) {
#pragma unroll
  for (int c = 0; c < 8; ++c)
    mine[lane * 8 + (c ^ (lane & 7))] =
        make_float4(acc[4 * c], acc[4 * c + 1], acc[4 * c + 2], acc[4 * c + 3]);
  __syncwarp();
}

// LATE: the residual is loaded here, half a block at a time, where registers are short.
template <typename T, int ACT, bool LATE = false>
__device__ __forceinline__ void write_staged(const ProductArgs& p, int split, const float4* mine,
                                             int64_t row0, int64_t col0, int lane,
                                             const ResidualBlock<T>& res) {
  const Epilogue& e = p.e;
  const int64_t col = col0 + (e.vec ? (lane & 7) * 4 : lane);
  const int rows = p.m - row0 < 32 ? static_cast<int>(p.m - row0) : 32;  // <= 0: none
  if (col < p.n && rows > 0) {
    if (e.partial) {
      float* out = e.partial + (split * p.m + row0) * p.n + col;
      if (e.vec) {
#pragma unroll 4
        for (int r = lane >> 3; r < rows; r += 4)
          *reinterpret_cast<float4*>(out + r * p.n) = mine[r * 8 + ((lane & 7) ^ (r & 7))];
      } else {
        const float* flat = reinterpret_cast<const float*>(mine);
#pragma unroll 4
        for (int r = 0; r < rows; ++r)
          out[r * p.n] = flat[r * 32 + (((lane >> 2) ^ (r & 7)) << 2) + (lane & 3)];
      }
    } else if (e.vec) {
      float bias[4];
      load_bias4<T>(e, col, p.n, bias);
      const int64_t at = (row0 + (lane >> 3)) * p.n + col;
      constexpr int kBatch = LATE ? 4 : 8;
#pragma unroll 1
      for (int i0 = 0; i0 < 8; i0 += kBatch) {
        Pack<T, 4> late[4];
        if constexpr (LATE) load_residual_part<T, 4>(p, row0, col0, lane, i0, late);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int r = (lane >> 3) + 4 * (i0 + i);
          if (r < rows) {
            const float4 f = mine[r * 8 + ((lane & 7) ^ (r & 7))];
            float v[4] = {f.x, f.y, f.z, f.w};
            Pack<T, 4> z{};
            finish4<T, ACT>(e, at + 4 * (i0 + i) * p.n, v, bias,
                            e.residual ? (LATE ? late[i & 3] : res.v[i]) : z);
          }
        }
      }
    } else {
      const float bias = e.bias ? to_float(static_cast<const T*>(e.bias)[col]) : 0.f;
      const float* flat = reinterpret_cast<const float*>(mine);
      float* preact = e.preact ? e.preact + row0 * p.n + col : nullptr;
      T* out = static_cast<T*>(e.out) + row0 * p.n + col;
      constexpr int kBatch = LATE ? 16 : 32;
#pragma unroll 1
      for (int i0 = 0; i0 < 32; i0 += kBatch) {
        Pack<T, 4> late[4];
        if constexpr (LATE) load_residual_part<T, 4>(p, row0, col0, lane, i0 / 4, late);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int r = i0 + i;
          if (r < rows) {
            const float v = flat[r * 32 + (((lane >> 2) ^ (r & 7)) << 2) + (lane & 3)] + bias;
            if (preact) preact[r * p.n] = v;
            float y = activate<ACT>(v, e.activation);
            if (e.residual)
              y += to_float(LATE ? late[(i / 4) & 3].v[i % 4] : res.v[i / 4].v[i % 4]);
            out[r * p.n] = from_float<T>(y);
          }
        }
      }
    }
  }
  __syncwarp();
}

template <typename T, int ACT>
__device__ __forceinline__ void write_block(const ProductArgs& p, int split, const float* acc,
                                            float4* mine, int64_t row0, int64_t col0, int lane,
                                            const ResidualBlock<T>& res) {
  stage_block(acc, mine, lane);
  write_staged<T, ACT>(p, split, mine, row0, col0, lane, res);
}

}  // namespace ictc
