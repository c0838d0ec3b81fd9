// Layer norm over the last dimension: forward, and backward with the reduction of the
// weight and bias gradients.
//
//   mean = sum x / C,  rstd = 1 / sqrt(sum (x - mean)^2 / C + eps),  u = (x - mean) rstd
//   y = u w + b
//   h = g w,  dx = rstd (h - mean(h) - u mean(h u)),  dw = sum_rows g u,  db = sum_rows g
//
// Both passes are bound by HBM: 2 (forward) or 3 (backward) values of the operand type
// move per element.  A row is read once and kept in registers, so the centred sum of
// squares is a second pass over registers and not over memory (no cancellation between
// sum x^2 and mean^2); it also sums the deviations themselves, which corrects the mean by
// what the first sum and 1 / C rounded away.  Narrow rows belong to up to 32 lanes of a warp that load them
// directly; wider rows to a whole CTA that takes them from a ring of shared-memory
// stages filled by bulk copies several rows ahead, because a CTA that loads, reduces and
// stores in turn leaves too few bytes in flight.  CTAs are persistent over rows: weights
// stay in registers, and the backward keeps each thread's columns of dw and db in
// registers over all of the CTA's rows and writes one partial row per CTA, summed in a
// fixed order by column_total_kernel.  Rows wider than a CTA's registers hold take the
// streaming kernels at the end, which read the row again for each pass.
//
// Measured: float32 1,048,576 x 64 forward 91 us (5.9 TB/s), backward 123 us (6.5 TB/s); bf16
// 16,384 x 4,096 forward 69 us (3.9 TB/s), backward 75 us (5.4 TB/s); float32 65,536 x 896
// forward 89 us (5.3 TB/s); f16 9,973 x 1,337 (no row on a 16-byte boundary) 50 and 38 us.
// The mean's correction is 7 of the 69 us.
#include <cuda_runtime.h>

#include <cstdint>
#include <initializer_list>

#include "common.cuh"
#include "dense_types.cuh"
#include "tma.cuh"

namespace ictc {
namespace {

// Threads of the widest CTA.  The backward holds five values per element (x, g, w, dw,
// db) where the forward holds three, so its CTA is half as large.
constexpr int kForwardThreads = 1024, kBackwardThreads = 512;
constexpr int kNarrowThreads = 128;
constexpr int kHeld = 16;  // elements of a row that one thread holds, at most
constexpr int kCodeRing = 22;  // bounded-wait code

// Sum over the threads of a row; every one of them gets the result.  `group` lanes of a
// warp (a power of two) use a butterfly, in which all add the same pairs; a whole CTA
// (`scratch` given: 32 values, zero past its warps) adds its warps' sums in warp order.
// Callers alternate between two scratch rows, so that one barrier per sum is enough.
__device__ __forceinline__ float group_sum(float v, int group, float* scratch) {
  const int width = scratch ? 32 : group;
  for (int o = width / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (scratch) {
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
    for (int w = 0; w < group / 32; w += 4) {
      const float4 q = *reinterpret_cast<const float4*>(scratch + w);
      v += (q.x + q.y) + (q.z + q.w);
    }
  }
  return v;
}

__device__ __forceinline__ float2 group_sum(float2 v, int group, float2* scratch) {
  if (!scratch) {
    for (int o = group / 2; o > 0; o >>= 1) {
      v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
      v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
  } else {
    // after one exchange the lower half warp adds x and the upper half y: five shuffles
    // instead of ten, the same pairs
    const int lane = threadIdx.x & 31;
    const bool upper = lane >= 16;
    float one = upper ? v.y : v.x;
    one += __shfl_xor_sync(0xffffffffu, upper ? v.x : v.y, 16);
    for (int o = 8; o > 0; o >>= 1) one += __shfl_xor_sync(0xffffffffu, one, o);
    if ((lane & 15) == 0) reinterpret_cast<float*>(scratch)[threadIdx.x >> 4] = one;
    __syncthreads();
    v = make_float2(0.f, 0.f);
    for (int w = 0; w < group / 32; w += 2) {
      const float4 q = *reinterpret_cast<const float4*>(scratch + w);
      v.x += q.x + q.z;
      v.y += q.y + q.w;
    }
  }
  return v;
}

// Paired arithmetic (one instruction for two elements).
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }

struct NormShape {
  int64_t rows, width;
  int64_t x_stride, g_stride;  // in elements; y and dx are contiguous
  int group;                   // threads per row
  float eps;
};

// V elements per access, N accesses per thread: thread t of a row's group holds columns
// (t + i * group) * V + j, i < N, j < V.  A width that is held in registers is below
// 2^14, so columns are ints; only row offsets need 64 bits.
template <typename T, int V, int N>
struct Held {
  Pack<T, V> v[N];
};

// Every thread's part of row r (nothing past the last row or column).
template <typename T, int V, int N>
__device__ __forceinline__ void load_row(const T* base, int64_t stride, int64_t r, bool in, int t,
                                         int group, int width, Held<T, V, N>& h) {
  const T* row = base + (in ? r : 0) * stride + t * V;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    h.v[i] = Pack<T, V>{};
    if (in && (t + i * group) * V < width)
      h.v[i] = *reinterpret_cast<const Pack<T, V>*>(row + i * group * V);
  }
}

// A thread's N V elements are handled as pairs, element 2 q and 2 q + 1; a single element
// (N = V = 1) is a pair with an empty half.
template <int V, int N>
constexpr int kPairs = (N * V + 1) / 2;

// Whether element e of the thread is a column.
template <int V>
__device__ __forceinline__ bool is_column(int e, int t, int group, int width) {
  return V > 1 ? (t + e / V * group) * V < width : t + e * group < width;
}

template <typename P, int V, int N>
__device__ __forceinline__ void load_params(const P* p, float missing, int t, int group, int width,
                                            float2 (&out)[kPairs<V, N>]) {
#pragma unroll
  for (int e = 0; e < 2 * kPairs<V, N>; ++e) {
    const int c = (t + e / V * group) * V + e % V;
    const float value = e < N * V && c < width ? (p ? to_float(p[c]) : missing) : 0.f;
    if (e & 1) out[e / 2].y = value;
    else out[e / 2].x = value;
  }
}

// Pair q of a held row.
template <typename T, int V, int N>
__device__ __forceinline__ float2 pair_of(const Held<T, V, N>& h, int q) {
  const int e = 2 * q, f = 2 * q + 1;
  return make_float2(to_float(h.v[e / V].v[e % V]),
                     f < N * V ? to_float(h.v[f / V].v[f % V]) : 0.f);
}

// v - mean, zero where there is no column (v is zero there).
template <int V>
__device__ __forceinline__ float2 centred(float2 v, float2 minus_mean, int q, int t, int group,
                                          int width) {
  float2 d = add2(v, minus_mean);
  if (!is_column<V>(2 * q, t, group, width)) d.x = 0.f;
  if (!is_column<V>(2 * q + 1, t, group, width)) d.y = 0.f;
  return d;
}

// This thread's share of (sum d, sum d^2), d = v - mean.
template <int V, int PAIRS>
__device__ __forceinline__ float2 deviation_sums(const float2 (&v)[PAIRS], float mean, int t,
                                                 int group, int width) {
  float2 sum = both(0.f), sq = both(0.f);
#pragma unroll
  for (int q = 0; q < PAIRS; ++q) {
    const float2 d = centred<V>(v[q], both(-mean), q, t, group, width);
    sum = add2(sum, d);
    sq = fma2(d, d, sq);
  }
  return make_float2(sum.x + sum.y, sq.x + sq.y);
}

// A row's statistics: u = (x - mean) rstd + shift.
struct Moments {
  float mean, rstd, shift;
};

// From a first mean and the row's sums about it.  A mean that is off by delta = sum d / C
// (1 / C is rounded, and so is the sum) would shift u by delta rstd: 0.9 for a constant row
// of 896 values of 1e5.  What mean + delta rounds away stays in `shift`.
__device__ __forceinline__ Moments moments_of(float first, float2 sums, float width, float inv,
                                              float eps) {
  const float delta = sums.x / width;
  float var = sums.y * inv - delta * delta;
  var = var < 0.f ? 0.f : var;  // a NaN stays
  Moments m;
  m.mean = first + delta;
  m.rstd = 1.f / sqrtf(var + eps);
  m.shift = ((m.mean - first) - delta) * m.rstd;
  return m;
}

template <typename T, int V, int N>
__device__ __forceinline__ float take_pairs(const Held<T, V, N>& row,
                                            float2 (&v)[kPairs<V, N>]) {
  float2 sum = both(0.f);
#pragma unroll
  for (int q = 0; q < kPairs<V, N>; ++q) {
    v[q] = pair_of(row, q);
    sum = add2(sum, v[q]);
  }
  return sum.x + sum.y;
}

// Stores the pairs o(q) of a row.
template <typename T, int V, int N, typename F>
__device__ __forceinline__ void store_row(T* row, int t, int group, int width, const F& o) {
  float2 p[kPairs<V, N>];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (t + i * group) * V;
    if (c < width) {
      Pack<T, V> pk;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int e = i * V + j;
        if (e % 2 == 0) p[e / 2] = o(e / 2);  // an odd column comes with its even one
        pk.v[j] = from_float<T>(e % 2 ? p[e / 2].y : p[e / 2].x);
      }
      *reinterpret_cast<Pack<T, V>*>(row + c) = pk;
    }
  }
}

template <typename T, int V, int N>
__device__ __forceinline__ void store_normed(T* row, const float2 (&v)[kPairs<V, N>],
                                             const float2 (&w)[kPairs<V, N>],
                                             const float2 (&b)[kPairs<V, N>],
                                             const Moments& m, int t, int group, int width) {
  store_row<T, V, N>(row, t, group, width, [&](int q) {
    return fma2(fma2(add2(v[q], both(-m.mean)), both(m.rstd), both(m.shift)), w[q], b[q]);
  });
}

// Adds a row to dw, db and returns this thread's share of (sum h, sum h u).  g and w are
// zero where there is no column.
template <typename T, int V, int N>
__device__ __forceinline__ float2 row_products(const Held<T, V, N>& px, const Held<T, V, N>& pg,
                                               const float2 (&w)[kPairs<V, N>],
                                               float2 (&dw)[kPairs<V, N>],
                                               float2 (&db)[kPairs<V, N>], float mean,
                                               float rstd) {
  float2 sh = both(0.f), shu = both(0.f);
#pragma unroll
  for (int q = 0; q < kPairs<V, N>; ++q) {
    const float2 g = pair_of(pg, q);
    const float2 u = mul2(add2(pair_of(px, q), both(-mean)), both(rstd));
    const float2 h = mul2(g, w[q]);
    dw[q] = fma2(g, u, dw[q]);
    db[q] = add2(db[q], g);
    sh = add2(sh, h);
    shu = fma2(h, u, shu);
  }
  return make_float2(sh.x + sh.y, shu.x + shu.y);
}

template <typename T, int V, int N>
__device__ __forceinline__ void store_gradient(T* row, const Held<T, V, N>& px,
                                               const Held<T, V, N>& pg,
                                               const float2 (&w)[kPairs<V, N>], float mean,
                                               float rstd, float mh, float mhu, int t, int group,
                                               int width) {
  store_row<T, V, N>(row, t, group, width, [&](int q) {
    const float2 u = mul2(add2(pair_of(px, q), both(-mean)), both(rstd));
    const float2 h = fma2(pair_of(pg, q), w[q], both(-mh));
    return mul2(both(rstd), fma2(u, both(-mhu), h));
  });
}

// The CTA's sums of dw and db to its rows of `partial` ([2][gridDim.x][width]): row groups
// joined in group order, one access column i at a time.
template <int V, int N>
__device__ __forceinline__ void store_columns(float* partial, float* column,
                                              const float2 (&dw)[kPairs<V, N>],
                                              const float2 (&db)[kPairs<V, N>], int t, int group,
                                              int width) {
  float* out_w = partial + static_cast<int64_t>(blockIdx.x) * width;
  float* out_b = out_w + static_cast<int64_t>(gridDim.x) * width;
  const int span = group * V, per_cta = blockDim.x / group;
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int e = i * V + j;
        const float2 p = half ? db[e / 2] : dw[e / 2];
        column[(threadIdx.x / group) * span + t * V + j] = e % 2 ? p.y : p.x;
      }
      __syncthreads();
      for (int k = threadIdx.x; k < span; k += blockDim.x) {
        const int c = i * span + k;
        if (c >= width) continue;
        float total = 0.f;
        for (int q = 0; q < per_cta; ++q) total += column[q * span + k];
        (half ? out_b : out_w)[c] = total;
      }
    }
}

// ---------------------------------------------------------- narrow rows: lanes of a warp

template <typename T, typename P, int V, int N>
__global__ void __launch_bounds__(kNarrowThreads, 8) norm_forward(
    const T* __restrict__ x, const P* __restrict__ weight, const P* __restrict__ bias,
    T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out, NormShape s) {
  const int group = s.group, width = static_cast<int>(s.width);
  const int t = threadIdx.x % group;
  const float inv = 1.f / static_cast<float>(width);
  float2 w[kPairs<V, N>], b[kPairs<V, N>];
  load_params<P, V, N>(weight, 1.f, t, group, width, w);
  load_params<P, V, N>(bias, 0.f, t, group, width, b);
  // Every lane runs the same number of rounds (the reductions are warp-wide); a round past
  // the last row loads and stores nothing.
  const int per_cta = kNarrowThreads / group;
  const int64_t step = static_cast<int64_t>(gridDim.x) * per_cta;
  int64_t base = static_cast<int64_t>(blockIdx.x) * per_cta;
  int64_t r = base + threadIdx.x / group;
  for (; base < s.rows; base += step, r += step) {
    Held<T, V, N> row;
    load_row<T, V, N>(x, s.x_stride, r, r < s.rows, t, group, width, row);
    float2 v[kPairs<V, N>];
    const float first = group_sum(take_pairs(row, v), group, nullptr) * inv;
    const Moments m =
        moments_of(first,
                   group_sum(deviation_sums<V>(v, first, t, group, width), group,
                             static_cast<float2*>(nullptr)),
                   static_cast<float>(width), inv, s.eps);
    if (r < s.rows) {
      store_normed<T, V, N>(y + r * width, v, w, b, m, t, group, width);
      if (t == 0 && mean_out != nullptr) {
        mean_out[r] = m.mean;
        rstd_out[r] = m.rstd;
      }
    }
  }
}

template <typename T, typename P, int V, int N>
__global__ void __launch_bounds__(kNarrowThreads, 4) norm_backward(
    const T* __restrict__ x, const P* __restrict__ weight, const float* __restrict__ mean_in,
    const float* __restrict__ rstd_in, const T* __restrict__ g, T* __restrict__ dx,
    float* __restrict__ partial, NormShape s) {
  __shared__ float column[kNarrowThreads * V];
  const int group = s.group, width = static_cast<int>(s.width);
  const int t = threadIdx.x % group;
  const float inv = 1.f / static_cast<float>(width);
  float2 w[kPairs<V, N>], dw[kPairs<V, N>], db[kPairs<V, N>];
  load_params<P, V, N>(weight, 1.f, t, group, width, w);
#pragma unroll
  for (int q = 0; q < kPairs<V, N>; ++q) dw[q] = db[q] = both(0.f);
  const int per_cta = kNarrowThreads / group;
  const int64_t step = static_cast<int64_t>(gridDim.x) * per_cta;
  int64_t base = static_cast<int64_t>(blockIdx.x) * per_cta;
  int64_t r = base + threadIdx.x / group;
  for (; base < s.rows; base += step, r += step) {
    const bool in = r < s.rows;
    Held<T, V, N> px, pg;
    load_row<T, V, N>(x, s.x_stride, r, in, t, group, width, px);
    load_row<T, V, N>(g, s.g_stride, r, in, t, group, width, pg);
    const float mean = in ? mean_in[r] : 0.f, rstd = in ? rstd_in[r] : 0.f;
    float2 sums = row_products(px, pg, w, dw, db, mean, rstd);
    if (dx != nullptr) {
      sums = group_sum(sums, group, static_cast<float2*>(nullptr));
      if (in)
        store_gradient<T, V, N>(dx + r * width, px, pg, w, mean, rstd, sums.x * inv, sums.y * inv,
                                t, group, width);
    }
  }
  if (partial != nullptr) store_columns<V, N>(partial, column, dw, db, t, group, width);
}

// ------------------------------------------------- wide rows: a CTA with a ring of stages
// Thread 0 fills a stage with the 16-byte blocks that cover a row (`shift` bytes of them
// come before it).  The tensor may not be read past its ends: a block that reaches over
// them is not copied, and the few elements in it are loaded where they are used.  A stage is free again once every thread has its part of
// the row in registers, which the next barrier of the reduction tells.

struct RowCopy {
  const char* from;   // first byte of the copied blocks
  uint32_t shift;     // of the row's first byte in the stage
  uint32_t bytes;     // copied
  int first, last;    // elements [first, last) of the row are in the stage
};

template <typename T>
__device__ __forceinline__ RowCopy row_copy(const T* base, int64_t stride, int64_t r, int64_t rows,
                                            int width) {
  const uintptr_t begin = reinterpret_cast<uintptr_t>(base + r * stride);
  const uintptr_t end = begin + static_cast<uintptr_t>(width) * sizeof(T);
  uintptr_t lo = begin & ~uintptr_t{15}, hi = (end + 15) & ~uintptr_t{15};
  RowCopy c;
  c.shift = static_cast<uint32_t>(begin - lo);
  c.first = 0;
  c.last = width;
  uint32_t skip = 0;
  if (lo < reinterpret_cast<uintptr_t>(base)) {
    lo += 16;
    skip = 16;
    c.first = static_cast<int>((lo - begin) / sizeof(T));
  }
  if (hi > reinterpret_cast<uintptr_t>(base + (rows - 1) * stride + width)) {
    hi -= 16;
    c.last = static_cast<int>((hi - begin) / sizeof(T));
  }
  c.from = reinterpret_cast<const char*>(lo);
  c.bytes = static_cast<uint32_t>(hi - lo);
  c.shift |= skip << 16;  // high half: where in the stage the copy goes
  return c;
}

template <typename T>
__device__ __forceinline__ uint32_t start_copy(unsigned char* stage, const T* base, int64_t stride,
                                               int64_t r, int64_t rows, int width, uint64_t* bar) {
  const RowCopy c = row_copy(base, stride, r, rows, width);
  bulk_g2s(stage + (c.shift >> 16), c.from, c.bytes, bar);
  return c.bytes;
}

// The thread's part of row r out of its stage.
template <typename T, int V, int N>
__device__ __forceinline__ void take_row(const unsigned char* stage, const T* base, int64_t stride,
                                         int64_t r, int64_t rows, int t, int group, int width,
                                         Held<T, V, N>& h) {
  if constexpr (V > 1) {  // every row is aligned: no shift, nothing outside the copy
    const T* row = reinterpret_cast<const T*>(stage);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (t + i * group) * V;
      h.v[i] = Pack<T, V>{};
      if (c < width) h.v[i] = *reinterpret_cast<const Pack<T, V>*>(row + c);
    }
  } else {
    const RowCopy rc = row_copy(base, stride, r, rows, width);
    const T* row = reinterpret_cast<const T*>(stage + (rc.shift & 0xffff));
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = t + i * group;
      h.v[i] = Pack<T, V>{};
      if (c < width) h.v[i].v[0] = row[c];
    }
    if (rc.first > 0 || rc.last < width) {  // a row at an end of the tensor
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int c = t + i * group;
        if (c < rc.first || (c >= rc.last && c < width)) h.v[i].v[0] = base[r * stride + c];
      }
    }
  }
}

struct Ring {
  uint32_t stage_bytes;  // one row of one operand, a multiple of 16
  int stages;
};

// Rows of the operands in `from` through the ring.  Every thread keeps the current stage
// and the parity of its barrier; fill(i, r) (thread 0; for a refill behind a barrier after
// the stage's row was taken) starts the copies of row r into stage i.
template <typename T, int OPERANDS>
struct RowRing {
  unsigned char* stages;
  uint64_t* full;
  Ring ring;
  const T* from[OPERANDS];
  int64_t stride[OPERANDS];
  int64_t rows;
  int width;
  int at;          // current stage
  uint32_t parity;

  __device__ __forceinline__ unsigned char* stage(int i) const {
    return stages + i * OPERANDS * ring.stage_bytes;
  }
  __device__ __forceinline__ void fill(int i, int64_t r) const {
    if (r >= rows) return;
    uint32_t bytes = 0;
#pragma unroll
    for (int o = 0; o < OPERANDS; ++o)
      bytes += row_copy(from[o], stride[o], r, rows, width).bytes;
    mbar_arrive_expect_tx(&full[i], bytes);
#pragma unroll
    for (int o = 0; o < OPERANDS; ++o)
      start_copy(stage(i) + o * ring.stage_bytes, from[o], stride[o], r, rows, width, &full[i]);
  }
  __device__ __forceinline__ bool wait() const { return mbar_wait(&full[at], parity, kCodeRing); }
  __device__ __forceinline__ void advance() {
    if (++at == ring.stages) {
      at = 0;
      parity ^= 1;
    }
  }
  // Thread 0, after a wait ran out: copies in flight land before the CTA goes away.
  __device__ __forceinline__ void settle() const {
    const unsigned long long start = global_timer_ns();
    while (global_timer_ns() - start < kDrainLimitNs) {
    }
  }
};

template <typename T, int OPERANDS>
__device__ __forceinline__ void ring_start(RowRing<T, OPERANDS>& q, unsigned char* smem,
                                           const Ring& ring, int (&failed)[2]) {
  q.full = reinterpret_cast<uint64_t*>(smem);
  q.stages = smem + 128;  // up to 16 barriers
  q.ring = ring;
  q.at = 0;
  q.parity = 0;
  if (threadIdx.x == 0) {
    failed[0] = failed[1] = 0;
    for (int i = 0; i < ring.stages; ++i) mbar_init(&q.full[i], 1);
    fence_mbarrier_init();
    for (int i = 0; i < ring.stages; ++i)
      q.fill(i, blockIdx.x + static_cast<int64_t>(i) * gridDim.x);
  }
  __syncthreads();
}

template <typename T, typename P, int V, int N>
__global__ void __launch_bounds__(kForwardThreads) norm_forward_ring(
    const T* __restrict__ x, const P* __restrict__ weight, const P* __restrict__ bias,
    T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out, NormShape s,
    Ring ring) {
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(16) float sums[32];
  __shared__ __align__(16) float2 deviations[32];
  __shared__ int failed[2];  // by the row's parity: a fast thread may be a row ahead
  const int group = blockDim.x, width = static_cast<int>(s.width), t = threadIdx.x;
  const float inv = 1.f / static_cast<float>(width);
  RowRing<T, 1> q;
  q.from[0] = x;
  q.stride[0] = s.x_stride;
  q.rows = s.rows;
  q.width = width;
  if (t < 32) {
    sums[t] = 0.f;
    deviations[t] = both(0.f);
  }
  ring_start(q, smem, ring, failed);
  float2 w[kPairs<V, N>], b[kPairs<V, N>];
  load_params<P, V, N>(weight, 1.f, t, group, width, w);
  load_params<P, V, N>(bias, 0.f, t, group, width, b);
  const int64_t ahead = static_cast<int64_t>(ring.stages) * gridDim.x;
  int k = 0;  // the row's parity
  bool gone = false;
  for (int64_t r = blockIdx.x; r < s.rows; r += gridDim.x, k ^= 1, q.advance()) {
    if (!q.wait()) failed[k] = 1;
    Held<T, V, N> row;
    take_row<T, V, N>(q.stage(q.at), x, s.x_stride, r, s.rows, t, group, width, row);
    float2 v[kPairs<V, N>];
    const float first = group_sum(take_pairs(row, v), group, sums) * inv;
    gone = failed[k] != 0;  // written before the barrier in group_sum: all threads agree
    if (gone) break;
    if (t == 0) q.fill(q.at, r + ahead);
    const Moments m = moments_of(
        first, group_sum(deviation_sums<V>(v, first, t, group, width), group, deviations),
        static_cast<float>(width), inv, s.eps);
    store_normed<T, V, N>(y + r * width, v, w, b, m, t, group, width);
    if (t == 0 && mean_out != nullptr) {
      mean_out[r] = m.mean;
      rstd_out[r] = m.rstd;
    }
  }
  if (gone && t == 0) q.settle();
}

template <typename T, typename P, int V, int N>
__global__ void __launch_bounds__(kBackwardThreads) norm_backward_ring(
    const T* __restrict__ x, const P* __restrict__ weight, const float* __restrict__ mean_in,
    const float* __restrict__ rstd_in, const T* __restrict__ g, T* __restrict__ dx,
    float* __restrict__ partial, NormShape s, Ring ring) {
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(16) float2 scratch[2][32];
  __shared__ int failed[2];  // by the row's parity: a fast thread may be a row ahead
  const int group = blockDim.x, width = static_cast<int>(s.width), t = threadIdx.x;
  const float inv = 1.f / static_cast<float>(width);
  RowRing<T, 2> q;
  q.from[0] = x;
  q.from[1] = g;
  q.stride[0] = s.x_stride;
  q.stride[1] = s.g_stride;
  q.rows = s.rows;
  q.width = width;
  if (t < 64) (&scratch[0][0])[t] = both(0.f);
  ring_start(q, smem, ring, failed);
  float2 w[kPairs<V, N>], dw[kPairs<V, N>], db[kPairs<V, N>];
  load_params<P, V, N>(weight, 1.f, t, group, width, w);
#pragma unroll
  for (int q = 0; q < kPairs<V, N>; ++q) dw[q] = db[q] = both(0.f);
  float next_mean = mean_in[blockIdx.x], next_rstd = rstd_in[blockIdx.x];
  const int64_t ahead = static_cast<int64_t>(ring.stages) * gridDim.x;
  int k = 0;  // the row's parity
  bool gone = false;
  for (int64_t r = blockIdx.x; r < s.rows; r += gridDim.x, k ^= 1, q.advance()) {
    const float mean = next_mean, rstd = next_rstd;
    const int64_t after = r + gridDim.x < s.rows ? r + gridDim.x : r;
    next_mean = mean_in[after];
    next_rstd = rstd_in[after];
    if (!q.wait()) failed[k] = 1;
    Held<T, V, N> px, pg;
    const unsigned char* stage = q.stage(q.at);
    take_row<T, V, N>(stage, x, s.x_stride, r, s.rows, t, group, width, px);
    take_row<T, V, N>(stage + ring.stage_bytes, g, s.g_stride, r, s.rows, t, group, width, pg);
    const float2 part = row_products(px, pg, w, dw, db, mean, rstd);
    const float2 sums = group_sum(part, group, scratch[k]);
    gone = failed[k] != 0;  // written before the barrier in group_sum: all threads agree
    if (gone) break;
    if (t == 0) q.fill(q.at, r + ahead);
    if (dx != nullptr)
      store_gradient<T, V, N>(dx + r * width, px, pg, w, mean, rstd, sums.x * inv, sums.y * inv, t,
                              group, width);
  }
  if (gone) {
    if (t == 0) q.settle();
    __syncthreads();
  }
  // every copy has landed and been read (or has settled): the stages are free
  if (partial != nullptr)
    store_columns<V, N>(partial, reinterpret_cast<float*>(smem + 128), dw, db, t, group, width);
}

// ------------------------------------------------ rows wider than a CTA's registers
// One CTA per row, three passes over the row (the second and third hit L2).

constexpr int kStreamThreads = 512;

template <typename T, typename P>
__global__ void __launch_bounds__(kStreamThreads) norm_forward_stream(
    const T* __restrict__ x, const P* __restrict__ weight, const P* __restrict__ bias,
    T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out, NormShape s) {
  __shared__ __align__(16) float sums[32];
  __shared__ __align__(16) float2 deviations[32];
  const float inv = 1.f / static_cast<float>(s.width);
  for (int64_t r = blockIdx.x; r < s.rows; r += gridDim.x) {
    const T* xr = x + r * s.x_stride;
    float sum = 0.f;
    for (int64_t c = threadIdx.x; c < s.width; c += kStreamThreads) sum += to_float(xr[c]);
    const float first = group_sum(sum, kStreamThreads, sums) * inv;
    float2 about = both(0.f);
    for (int64_t c = threadIdx.x; c < s.width; c += kStreamThreads) {
      const float d = to_float(xr[c]) - first;
      about.x += d;
      about.y += d * d;
    }
    const Moments m = moments_of(first, group_sum(about, kStreamThreads, deviations),
                                 static_cast<float>(s.width), inv, s.eps);
    for (int64_t c = threadIdx.x; c < s.width; c += kStreamThreads) {
      const float w = weight ? to_float(weight[c]) : 1.f, b = bias ? to_float(bias[c]) : 0.f;
      const float u = fmaf(to_float(xr[c]) - m.mean, m.rstd, m.shift);
      y[r * s.width + c] = from_float<T>(fmaf(u, w, b));
    }
    if (threadIdx.x == 0 && mean_out != nullptr) {
      mean_out[r] = m.mean;
      rstd_out[r] = m.rstd;
    }
  }
}

template <typename T, typename P>
__global__ void __launch_bounds__(kStreamThreads) norm_backward_stream(
    const T* __restrict__ x, const P* __restrict__ weight, const float* __restrict__ mean_in,
    const float* __restrict__ rstd_in, const T* __restrict__ g, T* __restrict__ dx, NormShape s) {
  __shared__ __align__(16) float2 scratch[2][32];
  const float inv = 1.f / static_cast<float>(s.width);
  int phase = 0;
  for (int64_t r = blockIdx.x; r < s.rows; r += gridDim.x) {
    const T* xr = x + r * s.x_stride;
    const T* gr = g + r * s.g_stride;
    const float mean = mean_in[r], rstd = rstd_in[r];
    float2 sums = make_float2(0.f, 0.f);
    for (int64_t c = threadIdx.x; c < s.width; c += kStreamThreads) {
      const float h = to_float(gr[c]) * (weight ? to_float(weight[c]) : 1.f);
      sums.x += h;
      sums.y += h * ((to_float(xr[c]) - mean) * rstd);
    }
    sums = group_sum(sums, kStreamThreads, scratch[phase]);
    phase ^= 1;
    for (int64_t c = threadIdx.x; c < s.width; c += kStreamThreads) {
      const float h = to_float(gr[c]) * (weight ? to_float(weight[c]) : 1.f);
      const float u = (to_float(xr[c]) - mean) * rstd;
      dx[r * s.width + c] = from_float<T>(rstd * (h - sums.x * inv - u * (sums.y * inv)));
    }
  }
}

// Column sums of g u and g over the rows blockIdx.y, + gridDim.y, ...; a thread per column.
template <typename T>
__global__ void __launch_bounds__(256) norm_columns_stream(
    const T* __restrict__ x, const float* __restrict__ mean_in,
    const float* __restrict__ rstd_in, const T* __restrict__ g, float* __restrict__ partial,
    NormShape s) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (c >= s.width) return;
  float dw = 0.f, db = 0.f;
  for (int64_t r = blockIdx.y; r < s.rows; r += gridDim.y) {
    const float gv = to_float(g[r * s.g_stride + c]);
    dw += gv * ((to_float(x[r * s.x_stride + c]) - mean_in[r]) * rstd_in[r]);
    db += gv;
  }
  partial[blockIdx.y * s.width + c] = dw;
  partial[(static_cast<int64_t>(gridDim.y) + blockIdx.y) * s.width + c] = db;
}

// ---------------------------------------------------------------------- host side

struct NormPlan {
  bool stream, wide;  // row too wide for registers; row for a whole CTA
  int vec, count;     // V and N
  int group, threads, grid;
  Ring ring;
  size_t smem;
};

constexpr size_t kRingBytes = 200 * 1024;  // shared memory of an SM that the rings may take

// The group is the smallest power of two that holds the row at kHeld elements a thread:
// more would push the backward (x, g, w, dw, db) past 128 registers, fewer would leave
// too little work behind each reduction.  Up to a warp's lanes the row is narrow; a wide
// row's CTA is as many warps as it needs.
NormPlan plan_norm(int64_t rows, int64_t width, int vec, size_t size, int device, bool backward) {
  NormPlan p{};
  p.vec = vec;
  const int64_t sms = sm_count(device);
  if (width > static_cast<int64_t>(backward ? kBackwardThreads : kForwardThreads) * kHeld) {
    p.stream = true;
    p.threads = kStreamThreads;
    p.grid = static_cast<int>(rows < sms * 4 ? rows : sms * 4);
    return p;
  }
  const int64_t units = ceil_div(width, vec);
  const int most = kHeld / vec;
  int group = 1;
  while (static_cast<int64_t>(group) * most < units) group *= 2;
  p.wide = group > 32;
  if (p.wide) group = static_cast<int>(32 * ceil_div(units, 32 * most));
  int count = 1;
  while (static_cast<int64_t>(group) * count < units) count *= 2;
  p.group = group;
  p.count = count;
  if (!p.wide) {
    p.threads = kNarrowThreads;
    const int64_t want = ceil_div(rows, p.threads / group);
    const int64_t cap = sms * (backward ? 4 : 16);
    p.grid = static_cast<int>(want < cap ? want : cap);
    return p;
  }
  // CTAs per SM by registers: 64 (forward) or 128 (backward) for each thread
  p.threads = group;
  const int64_t per_sm = (backward ? kBackwardThreads : kForwardThreads) / group;
  p.grid = static_cast<int>(rows < sms * per_sm ? rows : sms * per_sm);
  p.ring.stage_bytes = static_cast<uint32_t>(align_up(static_cast<size_t>(width) * size + 15, 16));
  const size_t row_bytes = p.ring.stage_bytes * (backward ? 2 : 1);
  int64_t stages = static_cast<int64_t>(kRingBytes / per_sm / row_bytes);
  stages = stages > 16 ? 16 : stages < 2 ? 2 : stages;
  p.ring.stages = static_cast<int>(stages);
  p.smem = 128 + stages * row_bytes;
  // the backward joins its columns in the same memory
  if (p.smem < 128 + static_cast<size_t>(group) * vec * sizeof(float))
    p.smem = 128 + static_cast<size_t>(group) * vec * sizeof(float);
  return p;
}

template <typename T, typename P>
struct NormArgs {
  const T* x;
  const P *weight, *bias;
  T* y;
  float *mean, *rstd;
  const T* g;
  T* dx;
  float* partial;
  NormShape s;
  NormPlan p;
  bool backward;
  cudaStream_t stream;
};

template <typename T, typename P, int V, int N>
int launch_norm(const NormArgs<T, P>& a) {
  const NormPlan& p = a.p;
  if (!p.wide) {
    if (!a.backward)
      norm_forward<T, P, V, N><<<p.grid, p.threads, 0, a.stream>>>(a.x, a.weight, a.bias, a.y,
                                                                   a.mean, a.rstd, a.s);
    else
      norm_backward<T, P, V, N><<<p.grid, p.threads, 0, a.stream>>>(
          a.x, a.weight, a.mean, a.rstd, a.g, a.dx, a.partial, a.s);
    return ICTC_OK;
  }
  if (!a.backward) {
    const auto kernel = norm_forward_ring<T, P, V, N>;
    const int st = allow_smem(reinterpret_cast<const void*>(kernel), p.smem);
    if (st != ICTC_OK) return st;
    kernel<<<p.grid, p.threads, p.smem, a.stream>>>(a.x, a.weight, a.bias, a.y, a.mean, a.rstd,
                                                    a.s, p.ring);
  } else {
    const auto kernel = norm_backward_ring<T, P, V, N>;
    const int st = allow_smem(reinterpret_cast<const void*>(kernel), p.smem);
    if (st != ICTC_OK) return st;
    kernel<<<p.grid, p.threads, p.smem, a.stream>>>(a.x, a.weight, a.mean, a.rstd, a.g, a.dx,
                                                    a.partial, a.s, p.ring);
  }
  return ICTC_OK;
}

template <typename T, typename P, int V>
int launch_norm_count(const NormArgs<T, P>& a) {
  switch (a.p.count) {
    case 1: return launch_norm<T, P, V, 1>(a);
    case 2: return launch_norm<T, P, V, 2>(a);
    case 4:
      if constexpr (V * 4 <= kHeld) return launch_norm<T, P, V, 4>(a);
      break;
    case 8:
      if constexpr (V * 8 <= kHeld) return launch_norm<T, P, V, 8>(a);
      break;
    case 16:
      if constexpr (V * 16 <= kHeld) return launch_norm<T, P, V, 16>(a);
      break;
  }
  return fail(ICTC_ERR_UNSUPPORTED, "layer norm: no kernel for this width");
}

template <typename T, typename P>
int launch_norm_vec(const NormArgs<T, P>& a) {
  constexpr int kFull = 16 / sizeof(T);
  return a.p.vec == kFull ? launch_norm_count<T, P, kFull>(a) : launch_norm_count<T, P, 1>(a);
}

// The widest access that every row of every operand starts on: 16 bytes or one element.
int vector_width(size_t size, int64_t width, int64_t s0, int64_t s1,
                 std::initializer_list<const void*> operands) {
  const int full = static_cast<int>(16 / size);
  bool ok = width % full == 0 && s0 % full == 0 && s1 % full == 0;
  for (const void* p : operands) ok = ok && aligned(p, 16);
  return ok ? full : 1;
}

int check_norm(int64_t rows, int64_t width, int32_t dtype, int32_t param_dtype) {
  if (rows < 0 || width < 1)
    return fail(ICTC_ERR_INVALID, "layer norm needs rows >= 0 and width >= 1, got %lld and %lld",
                static_cast<long long>(rows), static_cast<long long>(width));
  if (!known_dtype(dtype)) return fail(ICTC_ERR_INVALID, "unknown dtype code %d", dtype);
  if (param_dtype != dtype && param_dtype != ICTC_DTYPE_F32)
    return fail(ICTC_ERR_INVALID, "layer norm parameters must be float32 or the input's type");
  return ICTC_OK;
}

int current_device() {
  int device = 0;
  return cudaGetDevice(&device) == cudaSuccess ? device : 0;
}

template <typename T, typename P>
int run_forward(const void* x, int64_t x_stride, const void* weight, const void* bias, void* y,
                float* mean, float* rstd, int64_t rows, int64_t width, float eps,
                cudaStream_t stream) {
  NormArgs<T, P> a{};
  a.x = static_cast<const T*>(x);
  a.weight = static_cast<const P*>(weight);
  a.bias = static_cast<const P*>(bias);
  a.y = static_cast<T*>(y);
  a.mean = mean;
  a.rstd = rstd;
  a.stream = stream;
  const int vec = vector_width(sizeof(T), width, x_stride, 0, {x, y, weight, bias});
  a.p = plan_norm(rows, width, vec, sizeof(T), current_device(), false);
  a.s = {rows, width, x_stride, 0, a.p.group, eps};
  if (a.p.stream)
    norm_forward_stream<T, P><<<a.p.grid, kStreamThreads, 0, stream>>>(
        a.x, a.weight, a.bias, a.y, mean, rstd, a.s);
  else if (const int st = launch_norm_vec(a); st != ICTC_OK)
    return st;
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? ICTC_OK : cuda_fail(e, "layer norm forward launch");
}

// Partial rows of dw and db that a backward of this shape may write, over both access
// widths (the workspace does not depend on the pointers).
constexpr int64_t kStreamRowParts = 64;

int64_t norm_parts(int64_t rows, int64_t width, size_t size, int device) {
  int64_t most = 0;
  for (const int vec : {static_cast<int>(16 / size), 1}) {
    const NormPlan p = plan_norm(rows, width, vec, size, device, true);
    const int64_t parts = p.stream ? (rows < kStreamRowParts ? rows : kStreamRowParts) : p.grid;
    if (parts > most) most = parts;
  }
  return most;
}

template <typename T, typename P>
int run_backward(const void* x, int64_t x_stride, const void* weight, const float* mean,
                 const float* rstd, const void* g, int64_t g_stride, void* dx, void* dweight,
                 void* dbias, float* partial, int64_t rows, int64_t width, cudaStream_t stream) {
  NormArgs<T, P> a{};
  a.backward = true;
  a.x = static_cast<const T*>(x);
  a.weight = static_cast<const P*>(weight);
  a.mean = const_cast<float*>(mean);
  a.rstd = const_cast<float*>(rstd);
  a.g = static_cast<const T*>(g);
  a.dx = static_cast<T*>(dx);
  a.stream = stream;
  const bool columns = dweight != nullptr || dbias != nullptr;
  a.partial = columns ? partial : nullptr;
  const int vec = vector_width(sizeof(T), width, x_stride, g_stride, {x, g, dx, weight});
  a.p = plan_norm(rows, width, vec, sizeof(T), current_device(), true);
  a.s = {rows, width, x_stride, g_stride, a.p.group, 0.f};
  int64_t parts = a.p.grid;
  if (a.p.stream) {
    if (dx != nullptr)
      norm_backward_stream<T, P><<<a.p.grid, kStreamThreads, 0, stream>>>(
          a.x, a.weight, mean, rstd, a.g, a.dx, a.s);
    parts = rows < kStreamRowParts ? rows : kStreamRowParts;
    if (columns)
      norm_columns_stream<T><<<dim3(static_cast<unsigned>(ceil_div(width, 256)),
                                    static_cast<unsigned>(parts)),
                               256, 0, stream>>>(a.x, mean, rstd, a.g, partial, a.s);
  } else if (const int st = launch_norm_vec(a); st != ICTC_OK) {
    return st;
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "layer norm backward launch");
  if (columns) {
    const float* p0 = partial;
    const float* p1 = partial + parts * width;
    P* o0 = static_cast<P*>(dweight);
    P* o1 = static_cast<P*>(dbias);
    const unsigned halves = o0 != nullptr && o1 != nullptr ? 2 : 1;
    if (o0 == nullptr) {
      p0 = p1;
      o0 = o1;
    }
    column_total_kernel<P><<<dim3(static_cast<unsigned>(ceil_div(width, 32)), halves),
                             dim3(32, kColumnLanes), 0, stream>>>(p0, p1, o0, o1, parts, width);
    e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "layer norm column sum launch");
  }
  return ICTC_OK;
}

}  // namespace

int norm_take_device_error(int* code) {
  cudaError_t e;
  if (take_unit_device_error(code, &e) != 0) return cuda_fail(e, "layer norm device error flag");
  return ICTC_OK;
}

}  // namespace ictc

using namespace ictc;

extern "C" int32_t ictc_o2_layer_norm_forward(const void* x, int64_t x_stride, const void* weight,
                                              const void* bias, void* y, float* mean, float* rstd,
                                              int64_t rows, int64_t width, float eps,
                                              int32_t dtype, int32_t param_dtype, void* stream) {
  const int st = check_norm(rows, width, dtype, param_dtype);
  if (st != ICTC_OK) return st;
  if (!(eps >= 0.f)) return fail(ICTC_ERR_INVALID, "eps must be >= 0");
  if (rows == 0) return ICTC_OK;
  if (!x || !y || (mean == nullptr) != (rstd == nullptr))
    return fail(ICTC_ERR_INVALID, "null pointer");
  if (x_stride < 0) return fail(ICTC_ERR_INVALID, "negative row stride");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define ICTC_NORM_FORWARD(T, P) \
  return run_forward<T, P>(x, x_stride, weight, bias, y, mean, rstd, rows, width, eps, s)
  if (dtype == ICTC_DTYPE_F32) ICTC_NORM_FORWARD(float, float);
  if (dtype == ICTC_DTYPE_BF16) {
    if (param_dtype == ICTC_DTYPE_F32) ICTC_NORM_FORWARD(__nv_bfloat16, float);
    ICTC_NORM_FORWARD(__nv_bfloat16, __nv_bfloat16);
  }
  if (param_dtype == ICTC_DTYPE_F32) ICTC_NORM_FORWARD(__half, float);
  ICTC_NORM_FORWARD(__half, __half);
#undef ICTC_NORM_FORWARD
}

extern "C" int32_t ictc_o2_layer_norm_workspace(int64_t rows, int64_t width, int32_t dtype,
                                                int32_t device, size_t* bytes) {
  const int st = check_norm(rows, width, dtype, dtype);
  if (st != ICTC_OK) return st;
  if (!bytes) return fail(ICTC_ERR_INVALID, "null output");
  *bytes = static_cast<size_t>(2 * norm_parts(rows, width, dtype_size(dtype), device) * width) *
           sizeof(float);
  return ICTC_OK;
}

extern "C" int32_t ictc_o2_layer_norm_backward(
    const void* x, int64_t x_stride, const void* weight, const float* mean, const float* rstd,
    const void* grad_output, int64_t grad_stride, void* grad_x, void* grad_weight,
    void* grad_bias, void* workspace, size_t workspace_bytes, int64_t rows, int64_t width,
    int32_t dtype, int32_t param_dtype, void* stream) {
  const int st = check_norm(rows, width, dtype, param_dtype);
  if (st != ICTC_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    for (void* p : {grad_weight, grad_bias}) {
      if (!p) continue;
      const cudaError_t e =
          cudaMemsetAsync(p, 0, static_cast<size_t>(width) * dtype_size(param_dtype), s);
      if (e != cudaSuccess) return cuda_fail(e, "layer norm gradient clear");
    }
    return ICTC_OK;
  }
  if (!grad_x && !grad_weight && !grad_bias) return ICTC_OK;
  if (!x || !mean || !rstd || !grad_output) return fail(ICTC_ERR_INVALID, "null pointer");
  if (x_stride < 0 || grad_stride < 0) return fail(ICTC_ERR_INVALID, "negative row stride");
  if (grad_weight || grad_bias) {
    const size_t need =
        static_cast<size_t>(2 * norm_parts(rows, width, dtype_size(dtype), current_device()) *
                            width) * sizeof(float);
    if (!workspace || workspace_bytes < need)
      return fail(ICTC_ERR_WORKSPACE, "workspace has %zu bytes, needs %zu",
                  workspace ? workspace_bytes : 0, need);
  }
  float* partial = static_cast<float*>(workspace);
#define ICTC_NORM_BACKWARD(T, P)                                                              \
  return run_backward<T, P>(x, x_stride, weight, mean, rstd, grad_output, grad_stride, grad_x, \
                            grad_weight, grad_bias, partial, rows, width, s)
  if (dtype == ICTC_DTYPE_F32) ICTC_NORM_BACKWARD(float, float);
  if (dtype == ICTC_DTYPE_BF16) {
    if (param_dtype == ICTC_DTYPE_F32) ICTC_NORM_BACKWARD(__nv_bfloat16, float);
    ICTC_NORM_BACKWARD(__nv_bfloat16, __nv_bfloat16);
  }
  if (param_dtype == ICTC_DTYPE_F32) ICTC_NORM_BACKWARD(__half, float);
  ICTC_NORM_BACKWARD(__half, __half);
#undef ICTC_NORM_BACKWARD
}
