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


// One column of a row, v with the bias in it.
template <typename T>
__device__ __forceinline__ void store1(const Epilogue& e, int64_t row, int64_t col, int64_t n,
                                       float v) {
  if (e.preact) e.preact[row * n + col] = v;
  float y = activate(v, e.activation);
  if (e.residual) y += to_float(static_cast<const T*>(e.residual)[row * e.residual_stride + col]);
  static_cast<T*>(e.out)[row * n + col] = from_float<T>(y);
}

// Four columns of a row: bias, p, activation, residual and the store of y.
template <typename T>
__device__ __forceinline__ void finish4(const Epilogue& e, int64_t row, int64_t col, int64_t n,
                                        float (&v)[4], const float (&bias)[4]) {
  const int64_t at = row * n + col;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] += bias[j];
  if (e.vec) {
    if (e.preact) *reinterpret_cast<float4*>(e.preact + at) = make_float4(v[0], v[1], v[2], v[3]);
    Pack<T, 4> r{};
    if (e.residual)
      r = *reinterpret_cast<const Pack<T, 4>*>(static_cast<const T*>(e.residual) +
                                               row * e.residual_stride + col);
    Pack<T, 4> o;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      o.v[j] = from_float<T>(activate(v[j], e.activation) + (e.residual ? to_float(r.v[j]) : 0.f));
    *reinterpret_cast<Pack<T, 4>*>(static_cast<T*>(e.out) + at) = o;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col + j < n) store1<T>(e, row, col + j, n, v[j]);
  }
}

// One column of a row.
template <typename T>
__device__ __forceinline__ void finish1(const Epilogue& e, int64_t row, int64_t col, int64_t n,
                                        float v, float bias) {
  store1<T>(e, row, col, n, v + bias);
}

template <typename T>
__device__ __forceinline__ void load_bias4(const Epilogue& e, int64_t col, int64_t n,
                                           float (&bias)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    bias[j] = e.bias && col + j < n ? to_float(static_cast<const T*>(e.bias)[col + j]) : 0.f;
}


// One 32 x 32 block of an output tile, row-per-lane in `acc`, to memory: through the
// warp's 4 KB of shared memory (16-byte chunks XOR-swizzled by row), so that lanes of
// one row touch consecutive columns: eight lanes four columns each when the rows are
// aligned for that, 32 lanes one column each otherwise.  `redo` replaces a value (row,
// col, value) before it is used.
template <typename T, typename Redo>
__device__ __forceinline__ void write_block(const ProductArgs& p, int split, const float* acc,
                                            float4* mine, int64_t row0, int64_t col0, int lane,
                                            const Redo& redo) {
#pragma unroll
  for (int c = 0; c < 8; ++c)
    mine[lane * 8 + (c ^ (lane & 7))] =
        make_float4(acc[4 * c], acc[4 * c + 1], acc[4 * c + 2], acc[4 * c + 3]);
  __syncwarp();
  const Epilogue& e = p.e;
  if (e.vec) {
    const int64_t col = col0 + (lane & 7) * 4;
    if (col < p.n) {
      float bias[4];
      load_bias4<T>(e, col, p.n, bias);
#pragma unroll 4
      for (int i = 0; i < 8; ++i) {
        const int r = i * 4 + (lane >> 3);
        const int64_t row = row0 + r;
        if (row >= p.m) continue;
        const float4 f = mine[r * 8 + ((lane & 7) ^ (r & 7))];
        float v[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = redo(row, col + j, v[j]);
        if (e.partial)
          *reinterpret_cast<float4*>(e.partial + (split * p.m + row) * p.n + col) =
              make_float4(v[0], v[1], v[2], v[3]);
        else
          finish4<T>(e, row, col, p.n, v, bias);
      }
    }
  } else {
    const int64_t col = col0 + lane;
    if (col < p.n) {
      const float bias = e.bias ? to_float(static_cast<const T*>(e.bias)[col]) : 0.f;
      const float* flat = reinterpret_cast<const float*>(mine);
#pragma unroll 4
      for (int r = 0; r < 32; ++r) {
        const int64_t row = row0 + r;
        if (row >= p.m) break;
        const float v =
            redo(row, col, flat[r * 32 + (((lane >> 2) ^ (r & 7)) << 2) + (lane & 3)]);
        if (e.partial)
          e.partial[(split * p.m + row) * p.n + col] = v;
        else
          finish1<T>(e, row, col, p.n, v, bias);
      }
    }
  }
  __syncwarp();
}

}  // namespace ictc
