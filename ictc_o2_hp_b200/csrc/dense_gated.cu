// The gated linear layer y = act(pg) pu, (pg | pu) = x W^T + b, and its gradients.
//
//   pg = x Wg^T + bg,  pu = x Wu^T + bu,  y = act(pg) pu
//   x [M, K], W = (Wg; Wu) [2 H, K] (gate rows first), b [2 H], pg, pu and y [M, H]
//   du = g act(pg),  dg = g pu act'(pg),  D = (dg | du) [M, 2 H]
//   dx = D W,  dW = D^T x,  db = sum_rows D
//
// With both halves of W in one tensor the backward's products are those of a linear layer of
// 2 H outputs without activation (dense_linear.cu).
//
// Which kernel a forward takes:
//   up to 4 rows, aligned or small   FMAs, W read once (few_kernel)
//   up to 64 inputs and outputs,     one kernel per direction (dense_gated_narrow.cuh), which
//   contiguous 16-byte rows          keeps no p: the backward computes it again
//   16-bit, aligned rows             SM pairs fed by TMA (dense_pair.cuh, GATED)
//   float32, aligned rows            cut on the way in (dense_cut.cuh, GATED)
//   unaligned rows                   large products are copied to aligned rows first; for
//                                    small ones the linear layer leaves p in memory, and
//                                    gate_kernel makes y of it
// The backward forms D in a pass over p and g (gated_slope_kernel) but for the narrow layers.
// A tile of these kernels has the sums of both halves for the same columns of y, so that the
// epilogue needs nothing from another tile, and p is written only where a backward wants it.
//
// Relu's slope jumps at 0, where a p within its own rounding may have either sign.  In float32
// one such element among 10^8 moves dx and dW by 10^-4 of their norms, a thousand times what
// rounding does, so the sign is not left to the order in which a kernel happens to sum: p within
// the bounds of its error is computed again by fused multiply-adds in the order of k, bias last
// (settle_kernel; gated_narrow_backward_kernel for its own p), and every path has the same
// slopes.  (16-bit gradients are rounded by more than that.)
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "common.cuh"
#include "dense_cut.cuh"
#include "dense_epilogue.cuh"
#include "dense_gated_narrow.cuh"
#include "dense_pair.cuh"
#include "dense_plan.cuh"
#include "dense_thin.cuh"
#include "dense_types.cuh"
#include "tmap.cuh"

namespace ictc {
namespace {

// --------------------------------------------------------------------- y = act(pg) pu
// p is the sum of `splits` parts [m, 2 n], in order, and the bias; kept in `preact` where that is
// given.  One pass over what the products just left in L2 (2 to 4 us up to some megabytes).  V
// columns of each half a thread.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(256) gate_kernel(const float* parts, int splits,
                                                   const T* __restrict__ bias, float* preact,
                                                   T* __restrict__ y, int64_t m, int64_t n) {
  using Floats = Pack<float, V>;
  const int64_t units = n / V, total = m * units, part = m * 2 * n;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += step) {
    const int64_t row = i / units, col = (i - row * units) * V, at = row * 2 * n + col;
    Floats g = *reinterpret_cast<const Floats*>(parts + at);
    Floats u = *reinterpret_cast<const Floats*>(parts + at + n);
    for (int s = 1; s < splits; ++s) {
      const Floats a = *reinterpret_cast<const Floats*>(parts + s * part + at);
      const Floats b = *reinterpret_cast<const Floats*>(parts + s * part + at + n);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        g.v[j] += a.v[j];
        u.v[j] += b.v[j];
      }
    }
    if (bias) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        g.v[j] += to_float(bias[col + j]);
        u.v[j] += to_float(bias[n + col + j]);
      }
    }
    if (preact) {
      *reinterpret_cast<Floats*>(preact + at) = g;
      *reinterpret_cast<Floats*>(preact + at + n) = u;
    }
    Pack<T, V> o;
#pragma unroll
    for (int j = 0; j < V; ++j) o.v[j] = from_float<T>(activate<ACT>(g.v[j]) * u.v[j]);
    *reinterpret_cast<Pack<T, V>*>(y + row * n + col) = o;
  }
}

// ---------------------------------------------------------------- few rows: no tiles
// Blocks of up to four rows (blockIdx.y): W is read once a block and the products run on the
// FMA pipes.  `share` warps have one column of y, each a part of K; a lane reads V consecutive
// elements of both rows of W, and the warps' sums are added in warp order.  bf16 1 x 4,096 x
// 16,384: 49 us, 5.5 TB/s.
constexpr int kFewThreads = 256, kFewWarps = kFewThreads / 32;
constexpr int64_t kFewRows = 4;

template <typename T, int ROWS, int V>
__global__ void __launch_bounds__(kFewThreads) few_kernel(
    const T* __restrict__ x, int64_t ldx, const T* __restrict__ w, int64_t ldw, int64_t rows,
    int64_t n, int64_t k, int share, Epilogue e) {
  __shared__ float sums[kFewWarps][2 * ROWS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_cta = kFewWarps / share, part = warp % share;
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * ROWS;
  x += row0 * ldx;
  rows -= row0;
  if (e.preact) e.preact += row0 * 2 * n;
  T* y = static_cast<T*>(e.out) + row0 * n;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * per_cta; base < n;
       base += static_cast<int64_t>(gridDim.x) * per_cta) {
    const int64_t col = base + warp / share;
    float acc[2 * ROWS];
#pragma unroll
    for (int r = 0; r < 2 * ROWS; ++r) acc[r] = 0.f;
    if (col < n) {
      const T* wg = w + col * ldw;
      const T* wu = wg + n * ldw;
#pragma unroll 8
      for (int64_t c = (part * 32 + lane) * V; c < k; c += share * 32 * V) {
        const Pack<T, V> pg = *reinterpret_cast<const Pack<T, V>*>(wg + c);
        const Pack<T, V> pu = *reinterpret_cast<const Pack<T, V>*>(wu + c);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          if (r >= rows) break;
          const Pack<T, V> px = *reinterpret_cast<const Pack<T, V>*>(x + r * ldx + c);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float v = to_float(px.v[j]);
            acc[2 * r] = fmaf(v, to_float(pg.v[j]), acc[2 * r]);
            acc[2 * r + 1] = fmaf(v, to_float(pu.v[j]), acc[2 * r + 1]);
          }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < 2 * ROWS; ++r)
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], o);
    if (share > 1) {
      if (lane == 0)
#pragma unroll
        for (int r = 0; r < 2 * ROWS; ++r) sums[warp][r] = acc[r];
      __syncthreads();
      if (part == 0)
#pragma unroll
        for (int r = 0; r < 2 * ROWS; ++r) {
          acc[r] = 0.f;
          for (int q = 0; q < share; ++q) acc[r] += sums[warp + q][r];
        }
      __syncthreads();
    }
    if (part == 0 && lane == 0 && col < n) {
      const T* bias = static_cast<const T*>(e.bias);
      const float bg = bias ? to_float(bias[col]) : 0.f, bu = bias ? to_float(bias[n + col]) : 0.f;
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        if (r >= rows) break;
        const float pg = acc[2 * r] + bg, pu = acc[2 * r + 1] + bu;
        if (e.preact) {
          e.preact[r * 2 * n + col] = pg;
          e.preact[r * 2 * n + n + col] = pu;
        }
        y[r * n + col] = from_float<T>(activate<kAnyActivation>(pg, e.activation) * pu);
      }
    }
  }
}

// ------------------------------------------------- relu: p near 0, in the order of k
// A product's p and the sum in order differ by at most near_zero(k) |x|_2 |w|_2: the products
// that the cut parts drop, the tensor core's truncation (2.3 2^-24 of the sum so far a step of 16
// elements; sums are moved out every 256) and k rounding errors, seven standard deviations of
// them where that is less than all of one sign.
inline float near_zero(int64_t k) {
  const float elements = static_cast<float>(k);
  return 5.9604645e-8f * (6.f + 0.15f * fminf(elements, 256.f) + fminf(elements, 4.f * sqrtf(elements)));
}

// |w_c|_2 of the n gate rows of W, then |x_r|_2 of the m rows of x; `lanes` of a warp a row,
// kNormRows rows in flight.  Squares of finite values that leave float32's range are taken again
// in float64.
constexpr int kNormThreads = 256, kNormRows = 4;

template <int V>
__global__ void __launch_bounds__(kNormThreads)
    row_norm_kernel(const float* __restrict__ x, int64_t ldx, const float* __restrict__ w,
                    int64_t ldw, float* __restrict__ norms, int64_t m, int64_t n, int64_t k,
                    int lanes) {
  const int part = threadIdx.x % lanes, rows = kNormThreads / lanes;
  const int64_t total = m + n, step = static_cast<int64_t>(gridDim.x) * rows * kNormRows;
  const auto row_at = [&](int64_t r) { return r < n ? w + r * ldw : x + (r - n) * ldx; };
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * rows * kNormRows; base < total;
       base += step) {
    const int64_t r0 = base + threadIdx.x / lanes;
    const float* row[kNormRows];
    float sum[kNormRows], most[kNormRows];
#pragma unroll
    for (int q = 0; q < kNormRows; ++q) {
      row[q] = row_at(r0 + q * rows < total ? r0 + q * rows : 0);
      sum[q] = most[q] = 0.f;
    }
#pragma unroll 2
    for (int64_t c = part * V; c < k; c += lanes * V) {
      Pack<float, V> v[kNormRows];
#pragma unroll
      for (int q = 0; q < kNormRows; ++q) v[q] = *reinterpret_cast<const Pack<float, V>*>(row[q] + c);
#pragma unroll
      for (int q = 0; q < kNormRows; ++q)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          sum[q] = fmaf(v[q].v[j], v[q].v[j], sum[q]);
          most[q] = fmaxf(most[q], fabsf(v[q].v[j]));
        }
    }
#pragma unroll
    for (int q = 0; q < kNormRows; ++q)
      for (int o = lanes / 2; o > 0; o >>= 1) {
        sum[q] += __shfl_xor_sync(0xffffffffu, sum[q], o);
        most[q] = fmaxf(most[q], __shfl_xor_sync(0xffffffffu, most[q], o));
      }
#pragma unroll
    for (int q = 0; q < kNormRows; ++q) {
      if (part != 0 || r0 + q * rows >= total) continue;
      float norm = sqrtf(sum[q]);
      if ((sum[q] < 1e-30f || sum[q] > 1e38f) && most[q] > 0.f && most[q] <= 3.402823466e38f) {
        double wide = 0.0;
        for (int64_t c = 0; c < k; ++c) {
          const double v = row[q][c];
          wide = fma(v, v, wide);
        }
        norm = static_cast<float>(sqrt(wide));
      }
      norms[r0 + q * rows] = 1.01f * norm;
    }
  }
}

// Gate columns of preact that lie near 0 by fused multiply-adds in the order of k, bias last.
// One pass over the gate half, a run of segments a warp; what is near 0 in them then goes to a lane
// each.  float32 65,536 x 128 x 512, where that is 4 elements in 10^5: 11 us for the norms and 43;
// 4,096 x 16,384 x 2,048, 35 in 10^4 and long sums: 138 and 1,480 of a step's 12,600.
constexpr int kSettleWarps = 8, kSettleLoads = 8, kSettleRun = 32;

// V: elements of a load of preact, whose row lengths are whole ones; U: of x and W.  `run`
// segments a warp, kSettleRun at most.
template <int V, int U>
__global__ void __launch_bounds__(kSettleWarps * 32)
    settle_kernel(const float* __restrict__ x, int64_t ldx, const float* __restrict__ w,
                  int64_t ldw, const float* __restrict__ bias, const float* __restrict__ norms,
                  float* preact, int64_t m, int64_t n, int64_t k, float near, int run) {
  constexpr int kSegment = 32 * V * kSettleLoads, kRoom = 2 * kSegment;
  constexpr int kAhead = U == 4 ? 8 : 32;  // loads of x and of W in flight
  static_assert(kSegment * kSettleRun <= 65536);
  __shared__ uint16_t found[kSettleWarps][kRoom];
  __shared__ int counts[kSettleWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t total = m * n, length = static_cast<int64_t>(run) * kSegment;
  const int64_t next_row = 32 * V / n, next_col = 32 * V % n;  // a load of the warp on
  for (int64_t base = (static_cast<int64_t>(blockIdx.x) * kSettleWarps + warp) * length;
       base < total; base += static_cast<int64_t>(gridDim.x) * kSettleWarps * length) {
    if (lane == 0) counts[warp] = 0;
    __syncwarp();
    int64_t row = (base + lane * V) / n, col = base + lane * V - row * n;
#pragma unroll 1
    for (int segment = 0; segment < run; ++segment) {
      Pack<float, V> p[kSettleLoads];
      float size[kSettleLoads];
      int64_t cols[kSettleLoads];
#pragma unroll
      for (int i = 0; i < kSettleLoads; ++i) {
        size[i] = -1.f;
        cols[i] = col;
        if (row < m) {
          p[i] = *reinterpret_cast<const Pack<float, V>*>(preact + row * 2 * n + col);
          size[i] = near * norms[n + row];
        }
        row += next_row;
        col += next_col;
        if (col >= n) {
          col -= n;
          ++row;
        }
      }
      uint32_t mine = 0;
#pragma unroll
      for (int i = 0; i < kSettleLoads; ++i) {
        if (size[i] < 0.f) continue;
        const Pack<float, V> most = *reinterpret_cast<const Pack<float, V>*>(norms + cols[i]);
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (is_near(p[i].v[j], size[i] * most.v[j])) mine |= 1u << (i * V + j);
      }
      for (; mine != 0; mine &= mine - 1) {
        const int bit = __ffs(mine) - 1;
        found[warp][atomicAdd(&counts[warp], 1)] =
            static_cast<uint16_t>(segment * kSegment + (bit / V * 32 + lane) * V + bit % V);
      }
      __syncwarp();
      const int count = counts[warp];
      if (count <= kRoom - kSegment && segment + 1 < run) continue;
      for (int i = lane; i < count; i += 32) {
        const int64_t e = base + found[warp][i], r = e / n, c = e - r * n;
        const float* xr = x + r * ldx;
        const float* wr = w + c * ldw;
        float sum = 0.f;
#pragma unroll kAhead
        for (int64_t q = 0; q < k; q += U) {
          const Pack<float, U> a = *reinterpret_cast<const Pack<float, U>*>(xr + q);
          const Pack<float, U> b = *reinterpret_cast<const Pack<float, U>*>(wr + q);
#pragma unroll
          for (int j = 0; j < U; ++j) sum = fmaf(a.v[j], b.v[j], sum);
        }
        preact[r * 2 * n + c] = bias ? sum + bias[c] : sum;
      }
      __syncwarp();
      if (lane == 0) counts[warp] = 0;
      __syncwarp();
    }
  }
}

// ------------------------------------------------------- D = (dg | du) and its column sums
// Bound by HBM (bf16 16,384 x 4,096: 159 us, 5.9 TB/s; float32 65,536 x 512: 110 us, 6.1 TB/s;
// odd rows, f16 4,999 x 777, 18 us: issue).  A CTA owns a strip of columns of both halves and every gridDim.y-th block
// of rows; each thread keeps its columns' sums in registers, and the CTA's partial row of db
// is joined over its row lanes in order.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(256) gated_slope_kernel(
    const T* __restrict__ g, int64_t ldg, const float* __restrict__ p, T* __restrict__ d,
    int64_t ldd, float* __restrict__ partial, int64_t m, int64_t n, int lanes) {
  __shared__ float sums[2 * 256 * V];
  const int tx = threadIdx.x % lanes, ty = threadIdx.x / lanes, rows = 256 / lanes;
  const int64_t col = (static_cast<int64_t>(blockIdx.x) * lanes + tx) * V;
  float acc[2][V];
#pragma unroll
  for (int j = 0; j < V; ++j) acc[0][j] = acc[1][j] = 0.f;
  if (col < n) {
    constexpr int kAhead = V * sizeof(T) == 16 && sizeof(T) == 2 ? 2 : 4;  // rows in flight
    const int64_t step = static_cast<int64_t>(gridDim.y) * rows;
    for (int64_t r0 = static_cast<int64_t>(blockIdx.y) * rows + ty; r0 < m; r0 += kAhead * step) {
      Pack<T, V> pg[kAhead];
      Pack<float, V> gate[kAhead], up[kAhead];
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        const int64_t r = r0 + q * step;
        if (r < m) {
          pg[q] = *reinterpret_cast<const Pack<T, V>*>(g + r * ldg + col);
          gate[q] = *reinterpret_cast<const Pack<float, V>*>(p + r * 2 * n + col);
          up[q] = *reinterpret_cast<const Pack<float, V>*>(p + r * 2 * n + n + col);
        }
      }
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        const int64_t r = r0 + q * step;
        if (r >= m) break;
        Pack<T, V> dg, du;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float v = to_float(pg[q].v[j]);
          const float a = v * up[q].v[j] * activation_slope<ACT>(gate[q].v[j]);
          const float b = v * activate<ACT>(gate[q].v[j]);
          acc[0][j] += a;
          acc[1][j] += b;
          dg.v[j] = from_float<T>(a);
          du.v[j] = from_float<T>(b);
        }
        if (d != nullptr) {
          *reinterpret_cast<Pack<T, V>*>(d + r * ldd + col) = dg;
          *reinterpret_cast<Pack<T, V>*>(d + r * ldd + n + col) = du;
        }
      }
    }
  }
  if (partial == nullptr) return;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int j = 0; j < V; ++j) sums[((h * rows + ty) * lanes + tx) * V + j] = acc[h][j];
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * lanes * V; c += 256) {
    const int h = c / (lanes * V), in = c - h * lanes * V;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * lanes * V + in;
    if (at >= n) continue;
    float total = 0.f;
    for (int q = 0; q < rows; ++q) total += sums[(h * rows + q) * lanes * V + in];
    partial[blockIdx.y * 2 * n + h * n + at] = total;
  }
}

// ------------------------------------------------------------------- plan of a call

// What a call's pointers and strides allow.  (A single row may have any stride: the entry
// points take it as packed.)
int32_t layout_of(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t k, size_t size) {
  int32_t flags = 0;
  if (chunk_aligned(x, ldx, size) && chunk_aligned(w, ldw, size)) flags |= ICTC_LINEAR_ALIGNED;
  if (aligned(x, 16) && ldx == k) flags |= ICTC_LINEAR_PACKED;
  return flags;
}

// Products that the FMA pipes are through with before a tile's barriers, TMEM and tensor maps
// are set up: a warp for each column of four rows, and few rounds of them.  Float32 37 x 64 x
// 64 takes 3.6 us (narrow kernel 8.3), 256 x 64 x 64 6.1 (8.8), 512 x 64 x 64 8.8 (8.8), bf16 128
// x 64 x 64 3.9 (5.8), 256 x 64 x 64 6.6 (5.8), 16 x 512 x 512 4.9 (7.9), unaligned 300 x 33 x 77
// 6.1 (19.6 with the linear layer's kernels).
bool is_small(int64_t m, int64_t n, int64_t k, size_t size, bool whole) {
  const int64_t elements = whole ? 16 / static_cast<int64_t>(size) : 1;  // a lane's
  const int64_t warps = ceil_div(m, kFewRows) * n;
  return m <= 4096 && n <= 4096 && k <= 65536 &&
         warps <= (!whole ? 8192 : size == 4 ? 4096 : 2048) &&
         warps * ceil_div(k, 32 * elements) <= (whole ? 8192 : 16384);
}

// Layers whose backward computes p again at no cost of a pass (their g is contiguous too).
bool is_narrow(int64_t m, int64_t n, int64_t k, int dtype, int32_t layout) {
  const int64_t full = static_cast<int64_t>(16 / dtype_size(dtype));
  return (layout & ICTC_LINEAR_PACKED) && n <= kNarrow && k <= kNarrow && n % full == 0 &&
         k % full == 0 && m <= (1ll << 30);
}

enum class Way { few, narrow, pair, cut, general };

// Byte offsets of the workspace's parts, and its size.
struct GatedPlan {
  Way way;
  bool align;  // operands are copied to aligned rows
  PairPlan pair;
  Split cut;
  size_t x, w, partial;                  // forward
  size_t p, y;                           // forward, general
  size_t norms;                          // forward, where p is settled
  size_t d, columns, forward;            // backward
  size_t product, product_bytes, total;  // the linear layer's
};

struct Layout {
  size_t at = 0;
  size_t take(size_t bytes) {
    const size_t here = at;
    at += align_up(bytes, 256);
    return here;
  }
};

constexpr int64_t kSlopeParts = 296;

// Rows of copies and of D: whole 64-byte blocks.  Boxes of rows that begin between the 32-byte
// sectors of L2 fetch one more of them each (f16 4,999 x 1,112 x 776 forward 26.7 us, x 1,120
// 22.7).
constexpr int64_t kPitchUnit = 64;

int64_t row_pitch(int64_t width, size_t size) { return aligned_pitch(width, size, kPitchUnit); }

// Whether the p that a forward leaves for the backward is settled.
bool settles(int dtype, int activation) {
  return dtype == ICTC_DTYPE_F32 && activation == ICTC_ACT_RELU;
}

int plan_forward(int64_t m, int64_t n, int64_t k, int dtype, int activation, int32_t layout,
                 bool keep, int device, GatedPlan* b) {
  const size_t size = dtype_size(dtype);
  const bool rows_aligned = layout & ICTC_LINEAR_ALIGNED;
  const bool wide = dtype == ICTC_DTYPE_F32;
  Layout space;
  if (keep && settles(dtype, activation))
    b->norms = space.take(static_cast<size_t>(m + n) * sizeof(float));
  b->total = space.at;
  b->way = Way::general;
  const bool whole = rows_aligned && k % static_cast<int64_t>(16 / size) == 0;
  // three or four rows of 16 bits make more FMAs and conversions than the SM pairs' mostly empty
  // tiles cost (4 x 4,096 x 16,384 90 us, pairs 64; 4 x 2,048 x 2,048 10, pairs 13)
  const bool slow = size == 2 && m > 2 && n * k >= (1 << 24);
  if ((m <= kFewRows && (whole ? !slow : 2 * n * k <= (1 << 18))) ||
      is_small(m, n, k, size, whole)) {
    b->way = Way::few;
    return ICTC_OK;
  }
  if (!keep && is_narrow(m, n, k, dtype, layout)) {
    b->way = Way::narrow;
    return ICTC_OK;
  }
  // a few columns of both halves together: the linear layer's FMA kernels read x once, in any
  // layout, where tiles would be mostly empty (float32 40,000 x 732 x 4 64 us, tiles 74; x 733
  // 82, copied 110; aligned 16-bit tiles are as fast).  Likewise a few rows against weights off
  // the boundaries, which are not worth a copy.
  const bool thin =
      (2 * n <= kThin && k > kThin && (wide || !rows_aligned)) || (m <= kThin && !rows_aligned);
  b->align = !thin && !rows_aligned && worth_aligning(m, 2 * n, k);
  if (!thin && (rows_aligned || b->align)) {
    int splits = 0;
    if (wide) {
      b->cut = plan_product(m, 2 * n, k, true, device, 128, 128);
      if (b->cut.fits && m < (1ll << 30) && n < (1ll << 30) && k < (1ll << 30)) {
        b->way = Way::cut;
        splits = b->cut.splits;
      }
    } else {
      b->pair = plan_pair(m, 2 * n, k, device);
      if (b->pair.ok) {
        b->way = Way::pair;
        splits = b->pair.splits;
      }
    }
    if (b->way != Way::general) {
      if (b->align) {
        b->x = space.take(static_cast<size_t>(m) * row_pitch(k, size) * size);
        b->w = space.take(static_cast<size_t>(2 * n) * row_pitch(k, size) * size);
      }
      if (splits > 1) b->partial = space.take(static_cast<size_t>(splits) * m * 2 * n * sizeof(float));
      b->total = space.at;
      return ICTC_OK;
    }
  }
  // the sums by the linear layer of 2 n outputs: p, and in 16-bit types the layer's own
  // output, which nobody reads
  if (!keep) b->p = space.take(static_cast<size_t>(m) * 2 * n * sizeof(float));
  if (!wide) b->y = space.take(static_cast<size_t>(m) * 2 * n * size);
  size_t other;
  const int st = ictc_o2_linear_workspace(m, k, 2 * n, dtype, ICTC_ACT_NONE, layout, device,
                                          &b->product_bytes, &other);
  if (st != ICTC_OK) return st;
  b->product = space.take(b->product_bytes);
  b->total = space.at;
  return ICTC_OK;
}

// keep: the forward kept p.  Otherwise it is computed again, by the forward kernels where the
// layer is not narrow.
int plan_backward(int64_t m, int64_t n, int64_t k, int dtype, int activation, int32_t layout,
                  bool keep, int device, GatedPlan* b) {
  const size_t size = dtype_size(dtype);
  Layout space;
  if (!keep && is_narrow(m, n, k, dtype, layout)) {
    b->way = Way::narrow;
    b->partial = space.take(static_cast<size_t>(sm_count(device)) * 2 * n * (k + 1) * sizeof(float));
    b->total = space.at;
    return ICTC_OK;
  }
  if (!keep) {
    GatedPlan forward{};
    const int st = plan_forward(m, n, k, dtype, activation, layout, true, device, &forward);
    if (st != ICTC_OK) return st;
    b->p = space.take(static_cast<size_t>(m) * 2 * n * sizeof(float));
    b->y = space.take(static_cast<size_t>(m) * n * size);
    b->forward = space.take(forward.total);
  }
  b->way = Way::general;
  // the operands of both products: D as it is formed here, x and W copied where they need it
  const bool rows_aligned = layout & ICTC_LINEAR_ALIGNED;
  b->align = !rows_aligned && k > kThin && m > kThin && 2 * n > kThin &&
             worth_aligning(m, 2 * n, k);
  const int64_t pitch = row_pitch(2 * n, size);
  b->d = space.take(static_cast<size_t>(m) * pitch * size);
  b->columns =
      space.take(static_cast<size_t>(m < kSlopeParts ? m : kSlopeParts) * 2 * n * sizeof(float));
  if (b->align) {
    b->x = space.take(static_cast<size_t>(m) * row_pitch(k, size) * size);
    b->w = space.take(static_cast<size_t>(2 * n) * row_pitch(k, size) * size);
  }
  const bool packed = pitch == 2 * n || m <= 1;  // D
  const auto add_product = [&](int32_t flags) {
    size_t other, bytes = 0;
    const int st = ictc_o2_linear_workspace(m, k, 2 * n, dtype, ICTC_ACT_NONE, flags, device,
                                            &other, &bytes);
    if (bytes > b->product_bytes) b->product_bytes = bytes;
    return st;
  };
  int st;
  if (b->align) {
    // the flags do not say which operand is off the boundaries: x may stay in rows of its own
    // distance or be copied to packed ones, which take other products
    st = add_product(ICTC_LINEAR_ALIGNED);
    if (st == ICTC_OK && packed) st = add_product(ICTC_LINEAR_ALIGNED | ICTC_LINEAR_PACKED);
  } else {
    st = add_product(layout & (packed ? ~0 : ~ICTC_LINEAR_PACKED));
  }
  if (st != ICTC_OK) return st;
  b->product = space.take(b->product_bytes);
  b->total = space.at;
  return ICTC_OK;
}

template <typename T>
int run_gate(const float* parts, int splits, const T* bias, float* preact, T* y, int64_t m,
             int64_t n, int activation, cudaStream_t stream) {
  const bool vec = n % 4 == 0 && aligned(y, 4 * sizeof(T)) && aligned(parts, 16) &&
                   aligned(preact, 16);
  const int64_t blocks = ceil_div(m * (vec ? n / 4 : n), 256);
  const int64_t cap = static_cast<int64_t>(sm_count(current_device())) * 8;
  const unsigned grid = static_cast<unsigned>(blocks < cap ? blocks : cap);
  for_activation(activation, [&](auto act) {
    const auto kernel = vec ? gate_kernel<T, 4, act.value> : gate_kernel<T, 1, act.value>;
    kernel<<<grid, 256, 0, stream>>>(parts, splits, bias, preact, y, m, n);
  });
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? ICTC_OK : cuda_fail(e, "gated linear gate launch");
}

template <typename T>
int run_slope(const T* g, int64_t ldg, const float* p, T* d, int64_t ldd, float* columns, T* db,
              int64_t m, int64_t n, int activation, cudaStream_t stream) {
  constexpr int kFull = 16 / sizeof(T);
  const bool vec = n % kFull == 0 && chunk_aligned(g, ldg, sizeof(T)) && aligned(p, 16);
  const int64_t units = ceil_div(n, vec ? kFull : 1);
  int lanes = 1;
  while (lanes < 32 && lanes < units) lanes *= 2;
  const int64_t x = ceil_div(units, lanes), row_blocks = ceil_div(m, 256 / lanes);
  int64_t y = ceil_div(static_cast<int64_t>(sm_count(current_device())) * 8, x);
  if (y > kSlopeParts) y = kSlopeParts;
  if (y > row_blocks) y = row_blocks;
  const dim3 grid(static_cast<unsigned>(x), static_cast<unsigned>(y));
  for_activation(activation, [&](auto act) {
    if (vec)
      gated_slope_kernel<T, kFull, act.value>
          <<<grid, 256, 0, stream>>>(g, ldg, p, d, ldd, db ? columns : nullptr, m, n, lanes);
    else
      gated_slope_kernel<T, 1, act.value>
          <<<grid, 256, 0, stream>>>(g, ldg, p, d, ldd, db ? columns : nullptr, m, n, lanes);
  });
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "gated linear slope launch");
  if (db) {
    column_total_kernel<T><<<dim3(static_cast<unsigned>(ceil_div(2 * n, 32))),
                             dim3(32, kColumnLanes), 0, stream>>>(columns, columns, db, db, y,
                                                                  2 * n);
    e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "gated linear column sum launch");
  }
  return ICTC_OK;
}

// Calls f with the activation that a launch's epilogue needs: partial sums have none.
template <typename F>
void for_epilogue(const ProductArgs& p, const F& f) {
  for_activation(p.e.partial ? ICTC_ACT_NONE : p.e.activation, f);
}

template <typename T, int V>
int run_few(const T* x, int64_t ldx, const T* w, int64_t ldw, const Epilogue& e, int64_t m,
            int64_t n, int64_t k, cudaStream_t stream) {
  const int64_t sms = sm_count(current_device());
  const int64_t blocks = ceil_div(m, kFewRows);
  // warps of a CTA share a column where there are few, each with work for all of its lanes
  int share = 1;
  while (share < kFewWarps && n * blocks * share < sms * 8 && 2 * share * 32 * V <= k) share *= 2;
  const int64_t want = ceil_div(n, kFewWarps / share);
  const dim3 grid(static_cast<unsigned>(want < sms * 8 ? want : sms * 8),
                  static_cast<unsigned>(blocks));
  const auto kernel = m == 1   ? few_kernel<T, 1, V>
                      : m == 2 ? few_kernel<T, 2, V>
                               : few_kernel<T, kFewRows, V>;
  kernel<<<grid, kFewThreads, 0, stream>>>(x, ldx, w, ldw, m, n, k, share, e);
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? ICTC_OK : cuda_fail(err, "gated linear few-row launch");
}

template <typename T, int BN>
int launch_pair(const OperandMaps& maps, const ProductArgs& p, cudaStream_t stream) {
  const int64_t total = static_cast<int64_t>(p.tiles_m) * p.tiles_n * p.splits;
  const int64_t pairs = sm_count(current_device()) / 2;
  const unsigned grid = static_cast<unsigned>(2 * (total < pairs ? total : pairs));
  int st = ICTC_OK;
  for_epilogue(p, [&](auto act) {
    const auto kernel = pair_product_kernel<T, false, false, BN, act.value, true>;
    st = allow_smem(reinterpret_cast<const void*>(kernel), kPairSmem<BN>);
    if (st == ICTC_OK) kernel<<<grid, kPairThreads, kPairSmem<BN>, stream>>>(maps, p);
  });
  return st;
}

int launch_cut(const OperandMaps& maps, const ProductArgs& p, cudaStream_t stream) {
  constexpr int BN = 128;
  const int64_t total = static_cast<int64_t>(p.tiles_m) * p.tiles_n * p.splits;
  const int64_t sms = sm_count(current_device());
  const unsigned grid = static_cast<unsigned>(total < sms ? total : sms);
  int st = ICTC_OK;
  for_epilogue(p, [&](auto act) {
    const auto kernel = cut_product_kernel<false, false, BN, act.value, true>;
    if (!cut_shares_fit<false, false, BN, act.value, true>()) {
      st = fail(ICTC_ERR_UNSUPPORTED,
                "float32 product: built with fewer than %d registers a thread",
                kCutLaunchRegisters);
      return;
    }
    st = allow_smem(reinterpret_cast<const void*>(kernel), kCutSmem<BN>);
    if (st == ICTC_OK) kernel<<<grid, kCutThreads, kCutSmem<BN>, stream>>>(maps, p);
  });
  return st;
}

template <typename T>
GatedNarrowArgs narrow_args(const T* x, const T* w, int64_t ldw, const void* bias, int64_t m,
                            int64_t n, int64_t k) {
  GatedNarrowArgs p{};
  p.x = x; p.w = w; p.bias = bias;
  p.m = m; p.ldw = ldw;
  p.n = static_cast<int>(n); p.k = static_cast<int>(k);
  p.tiles = static_cast<int>(ceil_div(m, kNarrowTile));
  return p;
}

// `out` [m, wide_out] is y or dx.
template <typename T>
int narrow_maps(const T* x, const T* g, const T* out, int64_t m, int64_t n, int64_t k,
                int64_t wide_out, GatedNarrowMaps* maps) {
  constexpr int kSize = sizeof(T);
  constexpr bool kBf16 = std::is_same_v<T, __nv_bfloat16>;
  const auto encode = [&](const T* base, int64_t width, CUtensorMap* map) {
    return base == nullptr ||
           encode_swizzled_map(base, kSize, kBf16, width, m, width * kSize, kNarrowTile, map) == 0;
  };
  if (encode(x, k, &maps->x) && encode(g, n, &maps->g) && encode(out, wide_out, &maps->out))
    return ICTC_OK;
  return fail(ICTC_ERR_UNSUPPORTED, "gated linear: no tensor map for these operands");
}

template <typename T>
int run_narrow_forward(const T* x, const T* w, int64_t ldw, const Epilogue& e, int64_t m, int64_t n,
                       int64_t k, cudaStream_t stream) {
  const GatedNarrowArgs p = narrow_args(x, w, ldw, e.bias, m, n, k);
  GatedNarrowMaps maps{};
  int st = narrow_maps<T>(x, nullptr, static_cast<const T*>(e.out), m, n, k, n, &maps);
  if (st != ICTC_OK) return st;
  const int sms = sm_count(current_device());
  for_activation(e.activation, [&](auto act) {
    const auto kernel = gated_narrow_forward_kernel<T, act.value>;
    st = allow_smem(reinterpret_cast<const void*>(kernel), kGatedForwardSmem<T>);
    if (st == ICTC_OK)
      kernel<<<p.tiles < sms ? p.tiles : sms, kGatedForwardThreads, kGatedForwardSmem<T>, stream>>>(
          maps, p);
  });
  if (st != ICTC_OK) return st;
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? ICTC_OK : cuda_fail(err, "narrow gated forward launch");
}

template <typename T>
int run_narrow_backward(const T* x, const T* w, int64_t ldw, const void* bias, const T* g, T* dx,
                        T* dw, T* db, float* partial, int64_t m, int64_t n, int64_t k,
                        int activation, cudaStream_t stream) {
  GatedNarrowArgs p = narrow_args(x, w, ldw, bias, m, n, k);
  p.g = g;
  p.near = near_zero(k);
  p.partial = dw || db ? partial : nullptr;
  p.e.out = dx;
  GatedNarrowMaps maps{};
  int st = narrow_maps<T>(x, g, dx, m, n, k, k, &maps);
  if (st != ICTC_OK) return st;
  const int sms = sm_count(current_device());
  const int grid = p.tiles < sms ? p.tiles : sms;
  for_activation(activation, [&](auto act) {
    const auto kernel = gated_narrow_backward_kernel<T, act.value>;
    static const bool shares_fit = [&] {
      cudaFuncAttributes a{};
      return cudaFuncGetAttributes(&a, kernel) == cudaSuccess &&
             a.numRegs >= kBackLaunchRegisters;
    }();
    if (!shares_fit) {
      st = fail(ICTC_ERR_UNSUPPORTED, "gated linear: built with fewer than %d registers a thread",
                kBackLaunchRegisters);
      return;
    }
    st = allow_smem(reinterpret_cast<const void*>(kernel), kGatedBackwardSmem<T>);
    if (st == ICTC_OK) kernel<<<grid, kBackThreads, kGatedBackwardSmem<T>, stream>>>(maps, p);
  });
  if (st != ICTC_OK) return st;
  cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return cuda_fail(err, "narrow gated backward launch");
  if (!p.partial) return ICTC_OK;
  const int wide = 2 * p.n, nk = wide * p.k;
  narrow_total_kernel<T><<<static_cast<unsigned>(ceil_div(nk + wide, 32)), dim3(32, kColumnLanes),
                           0, stream>>>(partial, dw, db, grid, nk, wide);
  err = cudaGetLastError();
  return err == cudaSuccess ? ICTC_OK : cuda_fail(err, "narrow gated column sum launch");
}

template <typename T>
int run_tiles(const T* x, int64_t ldx, const T* w, int64_t ldw, Epilogue e, unsigned char* ws,
              const GatedPlan& plan, int64_t m, int64_t n, int64_t k, cudaStream_t stream) {
  int st = ICTC_OK;
  if (plan.align) {
    st = align_operand(&x, &ldx, m, k, ws + plan.x, stream, kPitchUnit);
    if (st == ICTC_OK) st = align_operand(&w, &ldw, 2 * n, k, ws + plan.w, stream, kPitchUnit);
    if (st != ICTC_OK) return st;
  }
  ProductArgs p{};
  p.m = m; p.n = n; p.k = k;
  OperandMaps maps;
  constexpr int kSize = sizeof(T);
  constexpr bool kBf16 = std::is_same_v<T, __nv_bfloat16>;
  int bn;
  if constexpr (kSize == 2) {
    p.tiles_m = plan.pair.tiles_m; p.tiles_n = plan.pair.tiles_n;
    p.splits = plan.pair.splits; p.chunks = plan.pair.chunks;
    p.chunks_per_split = plan.pair.chunks_per_split;
    bn = plan.pair.bn;
  } else {
    p.tiles_m = plan.cut.tiles_m; p.tiles_n = plan.cut.tiles_n;
    p.splits = plan.cut.splits; p.chunks = plan.cut.chunks;
    p.chunks_per_split = plan.cut.chunks_per_split;
    bn = plan.cut.bn;
  }
  constexpr int kBoxK = kSize == 2 ? 64 : kCutK;
  if (encode_matrix_map(x, kSize, kBf16, k, m, ldx * kSize, kBoxK, 128, &maps.a) != 0 ||
      encode_matrix_map(w, kSize, kBf16, k, 2 * n, ldw * kSize, kBoxK, bn / 2, &maps.b) != 0)
    return fail(ICTC_ERR_UNSUPPORTED, "gated linear: no tensor map for these operands");
  float* partial = p.splits > 1 ? reinterpret_cast<float*>(ws + plan.partial) : nullptr;
  e.vec = vec_epilogue<T>(e, n);
  p.e = e;
  p.e.partial = partial;
  if (partial) p.e.vec = n % 4 == 0;
  if constexpr (kSize == 2)
    st = bn == 256 ? launch_pair<T, 256>(maps, p, stream) : launch_pair<T, 128>(maps, p, stream);
  else
    st = launch_cut(maps, p, stream);
  if (st != ICTC_OK) return st;
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return cuda_fail(err, "gated linear product launch");
  if (!partial) return ICTC_OK;
  return run_gate<T>(partial, p.splits, static_cast<const T*>(e.bias), e.preact,
                     static_cast<T*>(e.out), m, n, e.activation, stream);
}

template <typename T>
int run_products(const void* x, int64_t ldx, const void* w, int64_t ldw, const Epilogue& e,
                 unsigned char* ws, const GatedPlan& plan, int64_t m, int64_t n, int64_t k,
                 int dtype, cudaStream_t stream) {
  const T* xt = static_cast<const T*>(x);
  const T* wt = static_cast<const T*>(w);
  if (plan.way == Way::few) {
    constexpr int kFull = 16 / sizeof(T);
    if (k % kFull == 0 && chunk_aligned(x, ldx, sizeof(T)) && chunk_aligned(w, ldw, sizeof(T)))
      return run_few<T, kFull>(xt, ldx, wt, ldw, e, m, n, k, stream);
    return run_few<T, 1>(xt, ldx, wt, ldw, e, m, n, k, stream);
  }
  if (plan.way == Way::narrow) return run_narrow_forward(xt, wt, ldw, e, m, n, k, stream);
  if (plan.way != Way::general) return run_tiles(xt, ldx, wt, ldw, e, ws, plan, m, n, k, stream);
  float* p = e.preact ? e.preact : reinterpret_cast<float*>(ws + plan.p);
  const bool wide = sizeof(T) == 4;
  const int st = ictc_o2_linear_forward(
      x, ldx, w, ldw, e.bias, nullptr, 0, wide ? static_cast<void*>(p) : ws + plan.y,
      wide ? nullptr : p, ws + plan.product, plan.product_bytes, m, k, 2 * n, dtype, ICTC_ACT_NONE,
      stream);
  if (st != ICTC_OK) return st;
  return run_gate<T>(p, 1, nullptr, nullptr, static_cast<T*>(e.out), m, n, e.activation, stream);
}

int run_settle(const float* x, int64_t ldx, const float* w, int64_t ldw, const Epilogue& e,
               float* norms, int64_t m, int64_t n, int64_t k, cudaStream_t stream) {
  const int64_t sms = sm_count(current_device());
  const auto grid = [&](int64_t blocks) {
    return static_cast<unsigned>(blocks < sms * 8 ? blocks : sms * 8);
  };
  const bool whole = k % 4 == 0 && chunk_aligned(x, ldx, 4) && chunk_aligned(w, ldw, 4);
  int lanes = 1;
  while (lanes < 32 && 4 * lanes * (whole ? 4 : 1) < k) lanes *= 2;  // four loads a lane
  const int64_t rows = kNormThreads / lanes * kNormRows;
  const auto norm = whole ? row_norm_kernel<4> : row_norm_kernel<1>;
  norm<<<grid(ceil_div(m + n, rows)), kNormThreads, 0, stream>>>(x, ldx, w, ldw, norms, m, n, k,
                                                                 lanes);
  cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return cuda_fail(err, "gated linear row norm launch");
  const bool vec = n % 4 == 0 && aligned(e.preact, 16);
  const auto settle = vec ? (whole ? settle_kernel<4, 4> : settle_kernel<4, 1>)
                          : (whole ? settle_kernel<1, 4> : settle_kernel<1, 1>);
  // one wave, if runs of kSettleRun segments make one
  const int64_t segments = ceil_div(m * n, 32 * kSettleLoads * (vec ? 4 : 1));
  const int64_t warps = sms * 3 * kSettleWarps;
  int64_t run = ceil_div(segments, warps);
  if (run > kSettleRun) run = kSettleRun;
  const int64_t blocks = ceil_div(segments, run * kSettleWarps);
  settle<<<grid(blocks), kSettleWarps * 32, 0, stream>>>(x, ldx, w, ldw,
                                                         static_cast<const float*>(e.bias), norms,
                                                         e.preact, m, n, k, near_zero(k),
                                                         static_cast<int>(run));
  err = cudaGetLastError();
  return err == cudaSuccess ? ICTC_OK : cuda_fail(err, "gated linear settle launch");
}

template <typename T>
int run_forward(const void* x, int64_t ldx, const void* w, int64_t ldw, const Epilogue& e,
                unsigned char* ws, const GatedPlan& plan, int64_t m, int64_t n, int64_t k,
                int dtype, cudaStream_t stream) {
  const int st = run_products<T>(x, ldx, w, ldw, e, ws, plan, m, n, k, dtype, stream);
  if (st != ICTC_OK || !e.preact || !settles(dtype, e.activation)) return st;
  return run_settle(static_cast<const float*>(x), ldx, static_cast<const float*>(w), ldw, e,
                    reinterpret_cast<float*>(ws + plan.norms), m, n, k, stream);
}

struct Backward {
  const void *x, *w, *bias;
  int64_t ldx, ldw;
  const float* preact;
  const void* g;
  int64_t ldg;
  void *dx, *dw, *db;
};

template <typename T>
int run_backward(const Backward& q, unsigned char* ws, const GatedPlan& plan, int64_t m, int64_t n,
                 int64_t k, int dtype, int activation, int32_t layout, cudaStream_t stream) {
  const T* g = static_cast<const T*>(q.g);
  T* db = static_cast<T*>(q.db);
  if (plan.way == Way::narrow)
    return run_narrow_backward(static_cast<const T*>(q.x), static_cast<const T*>(q.w), q.ldw, q.bias,
                               g, static_cast<T*>(q.dx), static_cast<T*>(q.dw), db,
                               reinterpret_cast<float*>(ws + plan.partial), m, n, k, activation,
                               stream);
  const float* p = q.preact;
  int st = ICTC_OK;
  if (!p) {
    GatedPlan forward{};
    st = plan_forward(m, n, k, dtype, activation, layout, true, current_device(), &forward);
    if (st != ICTC_OK) return st;
    Epilogue e{};
    e.bias = q.bias;
    e.preact = reinterpret_cast<float*>(ws + plan.p);
    e.out = ws + plan.y;
    e.activation = activation;
    p = e.preact;
    st = run_forward<T>(q.x, q.ldx, q.w, q.ldw, e, ws + plan.forward, forward, m, n, k, dtype,
                        stream);
    if (st != ICTC_OK) return st;
  }
  T* d = q.dx || q.dw ? reinterpret_cast<T*>(ws + plan.d) : nullptr;
  const int64_t pitch = row_pitch(2 * n, sizeof(T));
  st = run_slope<T>(g, q.ldg, p, d, pitch, reinterpret_cast<float*>(ws + plan.columns), db, m, n,
                    activation, stream);
  if (st != ICTC_OK || !d) return st;
  const T* x = static_cast<const T*>(q.x);
  const T* w = static_cast<const T*>(q.w);
  int64_t ldx = q.ldx, ldw = q.ldw;
  if (plan.align) {
    // (an operand that no product reads has its place all the same, for the layout's sake)
    const auto place = [&](const T** p, int64_t* ld, int64_t rows, size_t at, bool read) {
      if (st != ICTC_OK || chunk_aligned(*p, *ld, sizeof(T))) return;
      if (read) {
        st = align_operand(p, ld, rows, k, ws + at, stream, kPitchUnit);
      } else {
        *p = reinterpret_cast<const T*>(ws + at);
        *ld = row_pitch(k, sizeof(T));
      }
    };
    place(&x, &ldx, m, plan.x, q.dw != nullptr);
    place(&w, &ldw, 2 * n, plan.w, q.dx != nullptr);
    if (st != ICTC_OK) return st;
  }
  return ictc_o2_linear_backward(x, ldx, w, ldw, nullptr, d, pitch, q.dx, q.dw, nullptr,
                                 ws + plan.product, plan.product_bytes, m, k, 2 * n, dtype,
                                 ICTC_ACT_NONE, stream);
}

int check_gated(int64_t m, int64_t n, int64_t k, int32_t dtype, int32_t activation) {
  if (m < 0 || n < 1 || k < 1)
    return fail(ICTC_ERR_INVALID,
                "gated linear needs rows >= 0 and in, hidden >= 1, got %lld rows, in %lld, "
                "hidden %lld",
                static_cast<long long>(m), static_cast<long long>(k), static_cast<long long>(n));
  if (n > (1ll << 40) || k > (1ll << 40) || m > (1ll << 40))
    return fail(ICTC_ERR_UNSUPPORTED, "gated linear: a dimension is too large");
  if (!known_dtype(dtype)) return fail(ICTC_ERR_INVALID, "unknown dtype code %d", dtype);
  if (activation < ICTC_ACT_NONE || activation > ICTC_ACT_GELU_TANH)
    return fail(ICTC_ERR_INVALID, "unknown activation code %d", activation);
  return ICTC_OK;
}

int check_workspace(const void* workspace, size_t bytes, size_t needed) {
  if (needed > 0 && (!workspace || bytes < needed || !aligned(workspace, 256)))
    return fail(ICTC_ERR_WORKSPACE, "workspace has %zu bytes, needs %zu (256-byte aligned)",
                workspace ? bytes : 0, needed);
  return ICTC_OK;
}

}  // namespace

int gated_take_device_error(int* code) {
  cudaError_t e;
  if (take_unit_device_error(code, &e) != 0) return cuda_fail(e, "gated linear device error flag");
  return ICTC_OK;
}

}  // namespace ictc

using namespace ictc;

extern "C" int32_t ictc_o2_gated_linear_workspace(int64_t rows, int64_t in, int64_t hidden,
                                                  int32_t dtype, int32_t activation,
                                                  int32_t layout, int32_t keep, int32_t device,
                                                  size_t* forward_bytes, size_t* backward_bytes) {
  int st = check_gated(rows, hidden, in, dtype, activation);
  if (st != ICTC_OK) return st;
  if (!forward_bytes || !backward_bytes) return fail(ICTC_ERR_INVALID, "null output");
  *forward_bytes = *backward_bytes = 0;
  if (rows == 0) return ICTC_OK;
  GatedPlan forward{}, backward{};
  st = plan_forward(rows, hidden, in, dtype, activation, layout, keep != 0, device, &forward);
  if (st == ICTC_OK)
    st = plan_backward(rows, hidden, in, dtype, activation, layout, keep != 0, device, &backward);
  *forward_bytes = forward.total;
  *backward_bytes = backward.total;
  return st;
}

extern "C" int32_t ictc_o2_gated_linear_forward(const void* x, int64_t x_stride,
                                                const void* weight, int64_t weight_stride,
                                                const void* bias, void* y, float* preact,
                                                void* workspace, size_t workspace_bytes,
                                                int64_t rows, int64_t in, int64_t hidden,
                                                int32_t dtype, int32_t activation, void* stream) {
  int st = check_gated(rows, hidden, in, dtype, activation);
  if (st != ICTC_OK) return st;
  if (rows == 0) return ICTC_OK;
  if (!x || !weight || !y) return fail(ICTC_ERR_INVALID, "null pointer");
  if (rows == 1) x_stride = in;
  if (x_stride < in || weight_stride < in)
    return fail(ICTC_ERR_INVALID, "rows of x and weight must not overlap");
  const int32_t layout = layout_of(x, x_stride, weight, weight_stride, in, dtype_size(dtype));
  GatedPlan plan{};
  st = plan_forward(rows, hidden, in, dtype, activation, layout, preact != nullptr,
                    current_device(), &plan);
  if (st == ICTC_OK && plan.way == Way::narrow && !aligned(y, 16))
    st = fail(ICTC_ERR_INVALID, "without preact a narrow layer needs a 16-byte aligned y");
  if (st == ICTC_OK) st = check_workspace(workspace, workspace_bytes, plan.total);
  if (st != ICTC_OK) return st;
  Epilogue e{};
  e.bias = bias;
  e.preact = preact;
  e.out = y;
  e.activation = activation;
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define ICTC_GATED_FORWARD(T)                                                                 \
  return run_forward<T>(x, x_stride, weight, weight_stride, e, ws, plan, rows, hidden, in, dtype, \
                        s)
  if (dtype == ICTC_DTYPE_F32) ICTC_GATED_FORWARD(float);
  if (dtype == ICTC_DTYPE_BF16) ICTC_GATED_FORWARD(__nv_bfloat16);
  ICTC_GATED_FORWARD(__half);
#undef ICTC_GATED_FORWARD
}

extern "C" int32_t ictc_o2_gated_linear_backward(
    const void* x, int64_t x_stride, const void* weight, int64_t weight_stride, const void* bias,
    const float* preact, const void* grad_output, int64_t grad_stride, void* grad_x,
    void* grad_weight, void* grad_bias, void* workspace, size_t workspace_bytes, int64_t rows,
    int64_t in, int64_t hidden, int32_t dtype, int32_t activation, void* stream) {
  int st = check_gated(rows, hidden, in, dtype, activation);
  if (st != ICTC_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows == 0)
    return ictc_o2_linear_backward(nullptr, 0, nullptr, 0, nullptr, nullptr, 0, nullptr,
                                   grad_weight, grad_bias, nullptr, 0, 0, in, 2 * hidden, dtype,
                                   ICTC_ACT_NONE, stream);
  if (!grad_x && !grad_weight && !grad_bias) return ICTC_OK;
  if (!x || !weight || !grad_output) return fail(ICTC_ERR_INVALID, "null pointer");
  if (rows == 1) {
    x_stride = in;
    grad_stride = hidden;
  }
  if (x_stride < in || weight_stride < in)
    return fail(ICTC_ERR_INVALID, "rows of x and weight must not overlap");
  if (grad_stride < 0) return fail(ICTC_ERR_INVALID, "negative row stride");
  const size_t size = dtype_size(dtype);
  const int32_t layout = layout_of(x, x_stride, weight, weight_stride, in, size);
  if (!preact && is_narrow(rows, hidden, in, dtype, layout) &&
      (grad_stride != hidden || !aligned(grad_output, 16) || !aligned(grad_x, 16)))
    return fail(ICTC_ERR_INVALID,
                "without preact a narrow layer needs a contiguous grad_output, and it and grad_x "
                "16-byte aligned");
  GatedPlan plan{};
  st = plan_backward(rows, hidden, in, dtype, activation, layout, preact != nullptr,
                     current_device(), &plan);
  if (st == ICTC_OK) st = check_workspace(workspace, workspace_bytes, plan.total);
  if (st != ICTC_OK) return st;
  const Backward q{x, weight, bias, x_stride, weight_stride, preact, grad_output,
                   grad_stride, grad_x, grad_weight, grad_bias};
  unsigned char* ws = static_cast<unsigned char*>(workspace);
#define ICTC_GATED_BACKWARD(T) \
  return run_backward<T>(q, ws, plan, rows, hidden, in, dtype, activation, layout, s)
  if (dtype == ICTC_DTYPE_F32) ICTC_GATED_BACKWARD(float);
  if (dtype == ICTC_DTYPE_BF16) ICTC_GATED_BACKWARD(__nv_bfloat16);
  ICTC_GATED_BACKWARD(__half);
#undef ICTC_GATED_BACKWARD
}

extern "C" int32_t ictc_o2_gated_linear_keeps(int64_t rows, int64_t in, int64_t hidden,
                                              int32_t dtype, int32_t layout) {
  return known_dtype(dtype) && !is_narrow(rows, hidden, in, dtype, layout);
}
