// Products of the linear layer with a dimension of at most eight, in any layout: FMAs that
// read the one large operand once, where it lies.
//
// A tile of 64 or 128 columns would be mostly empty, and unaligned rows would be copied
// first; both cost several times the one pass over memory that such a product needs.  Which
// dimension of C[m, n] = sum over k of A(m, k) B(n, k) is small decides the form:
//   n (or m)      dot    rows of the other operand times a few staged in shared memory
//   k             outer  every element from at most eight products
//   n or m, with the other operand running along the rows of the sum:
//                 gram   columns of it, weighted by a few numbers a row, summed over the rows
// All sums are float32, in an order that does not depend on scheduling.
//
// Bound by HBM where few numbers meet each value of the large operand (dot, float32 7,245 x
// 14,302 x 1: 85 us, 4.9 TB/s), by the reads of the small operand beside it towards eight
// (dot, float32 136,107 x 175 x 6: 41 us; outer, float32 1,048,576 x 8 x 64 with SiLU: 101 us,
// 3.0 TB/s; the three products of a float16 training step of 7 x 4,826 x 9,305, rows off the
// boundaries: 53, 68 and 99 us for 90 MB each).  Calls that took tiles before: float32
// 937,427 x 89 x 6 forward 1,139 us (148 here), 343,990 x 65 x 7 407 us (52), 1 x 14,793 x
// 3,978 164 us (54).  Against the narrow kernel, which takes widths up to 64 otherwise (kernel
// times, SiLU, float32 and bf16): 37 x 8 x 64 4.5 and 3.6 us (narrow 6.8 and 6.0),
// 1,048,576 x 8 x 64 101 and 100 (151 and 114), x 64 x 8 90 and 87 (140 and 98), x 32 x 1 49
// and 16 (176 and 176).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "dense_epilogue.cuh"

namespace ictc {

constexpr int kThin = 8;                   // most of the small dimension
constexpr int kDotThreads = 512;
constexpr int kStripThreads = 256;
constexpr size_t kThinBytes = 192 * 1024;  // of shared memory for the staged operand

struct ThinArgs {
  const void* big;     // dot: [rows][len]; gram: [rows][width]
  int64_t big_ld;
  const void* small;   // element (i, c): i along k (dot), along the rows (outer, gram)
  int64_t small_i, small_c;
  const void* wide;    // outer: element (c, j)
  int64_t wide_c, wide_j;
  int64_t rows, width;
  int len, count;      // count <= kThin; outer and gram: their NC
  int lanes;           // outer, gram: threads along a row
  bool swapped;        // dot: C is [count][rows]; gram: [width][count]
  float* partial;      // gram: [gridDim.y][C]
  Epilogue e;
};

// Sums of N values over L lanes (t of them), each lane left with N / L of them (or one that
// L / N lanes share): every exchange halves what a lane still carries.  Returns the index
// of the lane's first value.
template <int N, int L>
__device__ __forceinline__ int scatter_sums(float (&v)[N], int t) {
  int index = 0;
#pragma unroll
  for (int o = L / 2, n = N; o > 0; o >>= 1) {
    if (n > 1) {
      n /= 2;
      const bool upper = t & o;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        if (i >= n) break;
        const float send = upper ? v[i] : v[i + n];
        v[i] = (upper ? v[i + n] : v[i]) + __shfl_xor_sync(0xffffffffu, send, o);
      }
      index += upper ? n : 0;
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    }
  }
  return index;
}

// dot: L lanes of a warp run along a row, V elements an access; a group of them holds R rows,
// and the staged operand's values serve all of them.
template <typename T, int V, int NC, int L, int R>
__global__ void __launch_bounds__(kDotThreads, 1) thin_dot_kernel(const __grid_constant__ ThinArgs p) {
  constexpr int G = 32 / L, N = R * NC;
  constexpr int U = (V > 1 ? 8 : 16) / R;  // accesses of a row in flight
  constexpr int kWarps = kDotThreads / 32;
  extern __shared__ __align__(16) float staged[];  // [NC][pitch]
  const int pitch = (p.len + 3) & ~3, len = p.len;
  const T* small = static_cast<const T*>(p.small);
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll 8
    for (int k = threadIdx.x; k < len; k += kDotThreads)
      staged[c * pitch + k] =
          c < p.count ? to_float(small[k * p.small_i + c * p.small_c]) : 0.f;
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = lane & (L - 1);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kWarps * G * R;
  for (int64_t base = (static_cast<int64_t>(blockIdx.x) * kWarps + warp) * G * R; base < p.rows;
       base += step) {
    const int64_t row0 = base + lane / L;
    const T* at[R];  // past the end: the last row again, its sums dropped
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = row0 + r * G;
      at[r] = static_cast<const T*>(p.big) + (row < p.rows ? row : p.rows - 1) * p.big_ld;
    }
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
    const auto meet = [&](const Pack<T, V>(&x)[R], int k) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const Pack<float, V> w = *reinterpret_cast<const Pack<float, V>*>(staged + c * pitch + k);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int j = 0; j < V; ++j)
            acc[r * NC + c] = fmaf(to_float(x[r].v[j]), w.v[j], acc[r * NC + c]);
      }
    };
    int k = t * V;
#pragma unroll 1
    for (; k + (U - 1) * L * V < len; k += U * L * V) {
      Pack<T, V> x[U][R];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int r = 0; r < R; ++r)
          x[u][r] = *reinterpret_cast<const Pack<T, V>*>(at[r] + k + u * L * V);
#pragma unroll
      for (int u = 0; u < U; ++u) meet(x[u], k + u * L * V);
    }
#pragma unroll 1
    for (; k < len; k += L * V) {
      Pack<T, V> x[R];
#pragma unroll
      for (int r = 0; r < R; ++r) x[r] = *reinterpret_cast<const Pack<T, V>*>(at[r] + k);
      meet(x, k);
    }
    __syncwarp();
    const int first = scatter_sums<N, L>(acc, t);
    if (L > N && (t & (L / N - 1)) != 0) continue;  // another lane has the same
#pragma unroll
    for (int i = 0; i < (N > L ? N / L : 1); ++i) {
      const int c = (first + i) % NC;
      const int64_t row = row0 + (first + i) / NC * G;
      if (c >= p.count || row >= p.rows) continue;
      const int64_t m = p.swapped ? c : row, n = p.swapped ? row : c;
      finish1<T, kAnyActivation>(p.e, m, n, p.swapped ? p.rows : p.count, acc[i],
                                 p.e.bias ? to_float(static_cast<const T*>(p.e.bias)[n]) : 0.f);
    }
  }
}

// The columns of a thread in a strip of `lanes` threads: V > 1 side by side, or kStrided
// of them `lanes` apart (rows off the boundaries).
constexpr int kStrided = 4;
template <int V>
constexpr int kColumns = V > 1 ? V : kStrided;

template <int V>
__device__ __forceinline__ int64_t strip_column(const ThinArgs& p, int tx, int j) {
  const int64_t base = static_cast<int64_t>(blockIdx.x) * p.lanes * kColumns<V>;
  return V > 1 ? base + tx * V + j : base + j * p.lanes + tx;
}

// outer: a thread keeps its columns' part of the wide operand in registers over all of its
// rows.
template <typename T, int V, int NC>
__global__ void __launch_bounds__(kStripThreads) thin_outer_kernel(const __grid_constant__ ThinArgs p) {
  constexpr int E = kColumns<V>, kAhead = 4;
  const int tx = threadIdx.x % p.lanes, ty = threadIdx.x / p.lanes;
  const int rows = kStripThreads / p.lanes;
  const T* wide = static_cast<const T*>(p.wide);
  const T* residual = static_cast<const T*>(p.e.residual);
  float w[NC][E], bias[E];
  bool in[E];
#pragma unroll
  for (int j = 0; j < E; ++j) {
    const int64_t col = strip_column<V>(p, tx, j);
    in[j] = col < p.width;
#pragma unroll
    for (int c = 0; c < NC; ++c)
      w[c][j] = in[j] ? to_float(wide[c * p.wide_c + col * p.wide_j]) : 0.f;
    bias[j] = p.e.bias && in[j] ? to_float(static_cast<const T*>(p.e.bias)[col]) : 0.f;
  }
  if (!in[0]) return;
  const int64_t col0 = strip_column<V>(p, tx, 0);
  const int64_t step = static_cast<int64_t>(gridDim.y) * rows;
  int64_t r = static_cast<int64_t>(blockIdx.y) * rows + ty;
  const auto some = [&](auto count) {
    constexpr int Q = count.value;
    float a[Q][NC];
    Pack<T, E> res[Q];
    const T* s = static_cast<const T*>(p.small) + r * p.small_i;
#pragma unroll
    for (int q = 0; q < Q; ++q, s += step * p.small_i)
#pragma unroll
      for (int c = 0; c < NC; ++c) a[q][c] = to_float(s[c * p.small_c]);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      res[q] = Pack<T, E>{};
      if (!residual) continue;
      const T* from = residual + (r + q * step) * p.e.residual_stride + col0;
      if constexpr (V > 1) {
        res[q] = *reinterpret_cast<const Pack<T, E>*>(from);
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (in[j]) res[q].v[j] = from[j * p.lanes];
      }
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int64_t at = (r + q * step) * p.width + col0;
      float v[E];
#pragma unroll
      for (int j = 0; j < E; ++j) {
        v[j] = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) v[j] = fmaf(a[q][c], w[c][j], v[j]);
      }
      if constexpr (V > 1) {
        finish4<T, kAnyActivation>(p.e, at, v, bias, res[q]);
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j) {
          if (!in[j]) break;
          const float sum = v[j] + bias[j];
          if (p.e.preact) p.e.preact[at + j * p.lanes] = sum;
          static_cast<T*>(p.e.out)[at + j * p.lanes] = from_float<T>(
              activate<kAnyActivation>(sum, p.e.activation) + to_float(res[q].v[j]));
        }
      }
    }
    r += Q * step;
  };
  while (r + (kAhead - 1) * step < p.rows) some(std::integral_constant<int, kAhead>{});
  while (r < p.rows) some(std::integral_constant<int, 1>{});
}

// gram: a CTA owns a strip of columns and every gridDim.y-th block of rows; a thread's sums
// stay in registers, and the CTA's part is joined over its row lanes in order.
template <typename T, int V, int NC>
__global__ void __launch_bounds__(kStripThreads) thin_gram_kernel(const __grid_constant__ ThinArgs p) {
  constexpr int E = kColumns<V>, kAhead = NC > 4 ? 2 : 4;
  __shared__ float sums[kStripThreads * E];
  const int tx = threadIdx.x % p.lanes, ty = threadIdx.x / p.lanes;
  const int rows = kStripThreads / p.lanes;
  const int64_t col0 = strip_column<V>(p, tx, 0);
  bool in[E];
  float acc[NC][E];
#pragma unroll
  for (int j = 0; j < E; ++j) {
    in[j] = strip_column<V>(p, tx, j) < p.width;
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[c][j] = 0.f;
  }
  if (in[0]) {
    const int64_t step = static_cast<int64_t>(gridDim.y) * rows;
    int64_t r = static_cast<int64_t>(blockIdx.y) * rows + ty;
    const auto some = [&](auto count) {
      constexpr int Q = count.value;
      Pack<T, E> x[Q];
      float a[Q][NC];
      const T* from = static_cast<const T*>(p.big) + r * p.big_ld + col0;
      const T* s = static_cast<const T*>(p.small) + r * p.small_i;
#pragma unroll
      for (int q = 0; q < Q; ++q, from += step * p.big_ld) {
        if constexpr (V > 1) {
          x[q] = *reinterpret_cast<const Pack<T, E>*>(from);
        } else {
          x[q] = Pack<T, E>{};
#pragma unroll
          for (int j = 0; j < E; ++j)
            if (in[j]) x[q].v[j] = from[j * p.lanes];
        }
      }
#pragma unroll
      for (int q = 0; q < Q; ++q, s += step * p.small_i)
#pragma unroll
        for (int c = 0; c < NC; ++c) a[q][c] = to_float(s[c * p.small_c]);
#pragma unroll
      for (int q = 0; q < Q; ++q)
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int j = 0; j < E; ++j) acc[c][j] = fmaf(a[q][c], to_float(x[q].v[j]), acc[c][j]);
      r += Q * step;
    };
    while (r + (kAhead - 1) * step < p.rows) some(std::integral_constant<int, kAhead>{});
    while (r < p.rows) some(std::integral_constant<int, 1>{});
  }
  const int strip = p.lanes * E;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * strip;
  float* out = p.partial + blockIdx.y * (p.width * NC);
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < E; ++j)
      sums[ty * strip + (V > 1 ? tx * V + j : j * p.lanes + tx)] = acc[c][j];
    __syncthreads();
    for (int i = threadIdx.x; i < strip && base + i < p.width; i += kStripThreads) {
      float total = 0.f;
      for (int q = 0; q < rows; ++q) total += sums[q * strip + i];
      out[p.swapped ? (base + i) * NC + c : c * p.width + base + i] = total;
    }
  }
}

}  // namespace ictc
