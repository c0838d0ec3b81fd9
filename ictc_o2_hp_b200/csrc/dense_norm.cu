// Layer norm over the last dimension: forward, and backward with the reduction of the
// weight and bias gradients.
//
//   mean = sum x / C,  rstd = 1 / sqrt(sum (x - mean)^2 / C + eps),  u = (x - mean) rstd
//   y = u w + b
//   h = g w,  dx = rstd (h - mean(h) - u mean(h u)),  dw = sum_rows g u,  db = sum_rows g
//
// Both passes are bound by HBM: 2 (forward) or 3 (backward) values of the operand type
// move per element.  A row belongs to a group of threads (a power of two, 4 lanes up to
// a whole CTA) that reads it once into registers, so the centred sum of squares is a
// second pass over registers and not over memory (no cancellation between sum x^2 and
// mean^2).  CTAs are persistent over rows: weights stay in registers, and the backward
// keeps each thread's columns of dw and db in registers over all of the CTA's rows and
// writes one partial row per CTA, summed in a fixed order by column_total_kernel.
// Rows wider than a CTA's registers hold take the streaming kernels at the end, which
// read the row again for each pass.
#include <cuda_runtime.h>

#include <cstdint>

#include "common.cuh"
#include "dense_types.cuh"

namespace ictc {
namespace {

// Threads of the widest row group.  The backward holds five values per element (x, g, w,
// dw, db) where the forward holds three, so its CTA is half as large.
constexpr int kForwardGroup = 1024, kBackwardGroup = 512;
constexpr int kHeld = 16;  // elements of a row that one thread holds, at most

// Sum over the `group` threads of a row; every one of them gets the result.  Groups up
// to a warp use a butterfly (every lane adds the same values in the same order); wider
// groups are the whole CTA and add the warps' sums in warp order.  Callers alternate
// between two scratch rows, so that one barrier per reduction is enough.
__device__ __forceinline__ float2 group_sum(float2 v, int group, float2* scratch) {
  const int width = group < 32 ? group : 32;
  for (int o = width / 2; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if (group > 32) {
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = make_float2(0.f, 0.f);
    for (int w = 0; w < group / 32; ++w) {
      v.x += scratch[w].x;
      v.y += scratch[w].y;
    }
  }
  return v;
}

struct NormShape {
  int64_t rows, width;
  int64_t x_stride, g_stride;  // in elements; y and dx are contiguous
  int group;                   // threads per row
  float eps;
};

// V elements per access, N accesses per thread: thread t of a row's group holds columns
// (t + i * group) * V + j, i < N, j < V.
template <typename T, typename P, int V, int N>
__global__ void __launch_bounds__(kForwardGroup) norm_forward(const T* __restrict__ x, const P* __restrict__ weight,
                             const P* __restrict__ bias, T* __restrict__ y,
                             float* __restrict__ mean_out, float* __restrict__ rstd_out,
                             NormShape s) {
  __shared__ float2 scratch[2][32];
  const int t = threadIdx.x % s.group;
  const int per_cta = blockDim.x / s.group;
  const float inv = 1.f / static_cast<float>(s.width);
  float w[N * V], b[N * V];
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int64_t c = static_cast<int64_t>(t + i * s.group) * V + j;
      const bool in = c < s.width;
      w[i * V + j] = in ? (weight ? to_float(weight[c]) : 1.f) : 0.f;
      b[i * V + j] = in && bias ? to_float(bias[c]) : 0.f;
    }
  // Every thread of the CTA runs the same number of rounds (the reductions meet at
  // warp and CTA barriers); a round past the last row loads and stores nothing.
  const int64_t step = static_cast<int64_t>(gridDim.x) * per_cta;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * per_cta;
  for (int64_t base = first; base < s.rows; base += step) {
    const int64_t r = base + threadIdx.x / s.group;
    const bool row_in = r < s.rows;
    const T* xr = x + r * s.x_stride;
    float v[N * V];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t c = static_cast<int64_t>(t + i * s.group) * V;
      Pack<T, V> pk{};
      if (row_in && c < s.width) pk = *reinterpret_cast<const Pack<T, V>*>(xr + c);
#pragma unroll
      for (int j = 0; j < V; ++j) v[i * V + j] = to_float(pk.v[j]);
    }
#pragma unroll
    for (int i = 0; i < N * V; ++i) sum += v[i];
    const float mean = group_sum(make_float2(sum, 0.f), s.group, scratch[0]).x * inv;
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bool in = static_cast<int64_t>(t + i * s.group) * V < s.width;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = v[i * V + j] - mean;
        v[i * V + j] = d;
        sq += in ? d * d : 0.f;
      }
    }
    const float var = group_sum(make_float2(sq, 0.f), s.group, scratch[1]).x * inv;
    const float rstd = 1.f / sqrtf(var + s.eps);
    if (row_in) {
      T* yr = y + r * s.width;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int64_t c = static_cast<int64_t>(t + i * s.group) * V;
        if (c < s.width) {
          Pack<T, V> pk;
#pragma unroll
          for (int j = 0; j < V; ++j)
            pk.v[j] = from_float<T>(v[i * V + j] * rstd * w[i * V + j] + b[i * V + j]);
          *reinterpret_cast<Pack<T, V>*>(yr + c) = pk;
        }
      }
      if (t == 0 && mean_out != nullptr) {
        mean_out[r] = mean;
        rstd_out[r] = rstd;
      }
    }
  }
}

// partial: [2][gridDim.x][width], the CTA's sums of g u and of g.
template <typename T, typename P, int V, int N>
__global__ void __launch_bounds__(kBackwardGroup) norm_backward(const T* __restrict__ x, const P* __restrict__ weight,
                              const float* __restrict__ mean_in,
                              const float* __restrict__ rstd_in, const T* __restrict__ g,
                              T* __restrict__ dx, float* __restrict__ partial, NormShape s) {
  extern __shared__ float column[];  // [per_cta][group * V] for the joining of dw and db
  __shared__ float2 scratch[2][32];
  const int t = threadIdx.x % s.group;
  const int per_cta = blockDim.x / s.group;
  const float inv = 1.f / static_cast<float>(s.width);
  float w[N * V], dw[N * V], db[N * V];
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int64_t c = static_cast<int64_t>(t + i * s.group) * V + j;
      w[i * V + j] = c < s.width ? (weight ? to_float(weight[c]) : 1.f) : 0.f;
      dw[i * V + j] = db[i * V + j] = 0.f;
    }
  const int64_t step = static_cast<int64_t>(gridDim.x) * per_cta;
  int phase = 0;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * per_cta; base < s.rows; base += step) {
    const int64_t r = base + threadIdx.x / s.group;
    const bool row_in = r < s.rows;
    Pack<T, V> px[N], pg[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t c = static_cast<int64_t>(t + i * s.group) * V;
      px[i] = Pack<T, V>{};
      pg[i] = Pack<T, V>{};
      if (row_in && c < s.width) {
        px[i] = *reinterpret_cast<const Pack<T, V>*>(x + r * s.x_stride + c);
        pg[i] = *reinterpret_cast<const Pack<T, V>*>(g + r * s.g_stride + c);
      }
    }
    const float mean = row_in ? mean_in[r] : 0.f, rstd = row_in ? rstd_in[r] : 0.f;
    float2 sums = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bool in = row_in && static_cast<int64_t>(t + i * s.group) * V < s.width;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float gv = to_float(pg[i].v[j]);
        const float u = (to_float(px[i].v[j]) - mean) * rstd;
        const float h = gv * w[i * V + j];
        if (in) {
          dw[i * V + j] += gv * u;
          db[i * V + j] += gv;
          sums.x += h;
          sums.y += h * u;
        }
      }
    }
    if (dx != nullptr) {
      sums = group_sum(sums, s.group, scratch[phase]);
      phase ^= 1;
      const float mh = sums.x * inv, mhu = sums.y * inv;
      if (row_in) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int64_t c = static_cast<int64_t>(t + i * s.group) * V;
          if (c < s.width) {
            Pack<T, V> pk;
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const float u = (to_float(px[i].v[j]) - mean) * rstd;
              const float h = to_float(pg[i].v[j]) * w[i * V + j];
              pk.v[j] = from_float<T>(rstd * (h - mh - u * mhu));
            }
            *reinterpret_cast<Pack<T, V>*>(dx + r * s.width + c) = pk;
          }
        }
      }
    }
  }
  if (partial == nullptr) return;
  // Join the CTA's row groups in group order, one access column i at a time.
  float* out_w = partial + static_cast<int64_t>(blockIdx.x) * s.width;
  float* out_b = out_w + static_cast<int64_t>(gridDim.x) * s.width;
  const int span = s.group * V;
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < V; ++j)
        column[(threadIdx.x / s.group) * span + t * V + j] =
            half ? db[i * V + j] : dw[i * V + j];
      __syncthreads();
      for (int k = threadIdx.x; k < span; k += blockDim.x) {
        const int64_t c = static_cast<int64_t>(i) * span + k;
        if (c >= s.width) continue;
        float total = 0.f;
        for (int q = 0; q < per_cta; ++q) total += column[q * span + k];
        (half ? out_b : out_w)[c] = total;
      }
    }
}

// ------------------------------------------------ rows wider than a CTA's registers
// One CTA per row, three passes over the row (the second and third hit L2).

constexpr int kStreamThreads = 512;

template <typename T, typename P>
__global__ void __launch_bounds__(kStreamThreads) norm_forward_stream(
    const T* __restrict__ x, const P* __restrict__ weight, const P* __restrict__ bias,
    T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out, NormShape s) {
  __shared__ float2 scratch[2][32];
  const float inv = 1.f / static_cast<float>(s.width);
  for (int64_t r = blockIdx.x; r < s.rows; r += gridDim.x) {
    const T* xr = x + r * s.x_stride;
    float sum = 0.f;
    for (int64_t c = threadIdx.x; c < s.width; c += kStreamThreads) sum += to_float(xr[c]);
    const float mean = group_sum(make_float2(sum, 0.f), kStreamThreads, scratch[0]).x * inv;
    float sq = 0.f;
    for (int64_t c = threadIdx.x; c < s.width; c += kStreamThreads) {
      const float d = to_float(xr[c]) - mean;
      sq += d * d;
    }
    const float var = group_sum(make_float2(sq, 0.f), kStreamThreads, scratch[1]).x * inv;
    const float rstd = 1.f / sqrtf(var + s.eps);
    for (int64_t c = threadIdx.x; c < s.width; c += kStreamThreads) {
      const float w = weight ? to_float(weight[c]) : 1.f, b = bias ? to_float(bias[c]) : 0.f;
      y[r * s.width + c] = from_float<T>((to_float(xr[c]) - mean) * rstd * w + b);
    }
    if (threadIdx.x == 0 && mean_out != nullptr) {
      mean_out[r] = mean;
      rstd_out[r] = rstd;
    }
  }
}

template <typename T, typename P>
__global__ void __launch_bounds__(kStreamThreads) norm_backward_stream(
    const T* __restrict__ x, const P* __restrict__ weight, const float* __restrict__ mean_in,
    const float* __restrict__ rstd_in, const T* __restrict__ g, T* __restrict__ dx, NormShape s) {
  __shared__ float2 scratch[2][32];
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

bool streams(int64_t width, bool backward) {
  return width > static_cast<int64_t>(backward ? kBackwardGroup : kForwardGroup) * kHeld;
}

struct NormPlan {
  bool stream;     // row too wide for registers
  int vec, count;  // V and N
  int group, threads, grid;
};

// A thread holds up to 16 elements of a row: more would push the backward (x, g, w, dw,
// db) past 128 registers, fewer would leave too few bytes in flight.  The group is the
// smallest power of two that holds the row that way, but at least as many lanes as make
// one 16-byte access each.
NormPlan plan_norm(int64_t rows, int64_t width, int vec, int device, bool backward) {
  NormPlan p{};
  p.vec = vec;
  if (streams(width, backward)) {
    p.stream = true;
    p.threads = kStreamThreads;
    const int64_t cap = static_cast<int64_t>(sm_count(device)) * 4;
    p.grid = static_cast<int>(rows < cap ? rows : cap);
    return p;
  }
  const int64_t units = ceil_div(width, vec);
  int most = kHeld / vec;
  if (most > 4 && vec > 1) most = 4;
  int group = 1;
  while (static_cast<int64_t>(group) * most < units) group *= 2;
  int count = 1;
  while (static_cast<int64_t>(group) * count < units) count *= 2;
  p.group = group;
  p.count = count;
  p.threads = group > 32 ? group : 128;  // a group wider than a warp is a whole CTA
  const int64_t per_cta = p.threads / group;
  const int64_t want = ceil_div(rows, per_cta);
  // The backward writes 2 x width floats per CTA, so its grid stays at what fills the
  // SMs; the forward may run more, shorter CTAs.
  const int64_t resident = backward ? (p.threads >= 512 ? 1024 / p.threads : 512 / p.threads)
                                    : 2048 / p.threads;
  const int64_t cap = static_cast<int64_t>(sm_count(device)) * (resident < 1 ? 1 : resident);
  p.grid = static_cast<int>(want < cap ? want : cap);
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
void launch_norm(const NormArgs<T, P>& a) {
  if (!a.backward)
    norm_forward<T, P, V, N><<<a.p.grid, a.p.threads, 0, a.stream>>>(a.x, a.weight, a.bias, a.y,
                                                                     a.mean, a.rstd, a.s);
  else
    norm_backward<T, P, V, N>
        <<<a.p.grid, a.p.threads, static_cast<size_t>(a.p.threads) * V * sizeof(float),
           a.stream>>>(a.x, a.weight, a.mean, a.rstd, a.g, a.dx, a.partial, a.s);
}

template <typename T, typename P, int V>
void launch_norm_count(const NormArgs<T, P>& a) {
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
}

template <typename T, typename P>
void launch_norm_vec(const NormArgs<T, P>& a) {
  constexpr int kFull = 16 / sizeof(T);
  if (a.p.vec == kFull) launch_norm_count<T, P, kFull>(a);
  else launch_norm_count<T, P, 1>(a);
}

// The widest access that every row of every operand starts on: 16 bytes or one element.
int vector_width(size_t size, int64_t width, int64_t s0, int64_t s1, const void* a, const void* b,
                 const void* c) {
  const int full = static_cast<int>(16 / size);
  const bool ok = width % full == 0 && s0 % full == 0 && s1 % full == 0 && aligned(a, 16) &&
                  aligned(b, 16) && aligned(c, 16);
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
  const int vec = vector_width(sizeof(T), width, x_stride, 0, x, y, nullptr);
  a.p = plan_norm(rows, width, vec, current_device(), false);
  a.s = {rows, width, x_stride, 0, a.p.group, eps};
  if (a.p.stream)
    norm_forward_stream<T, P><<<a.p.grid, kStreamThreads, 0, stream>>>(
        a.x, a.weight, a.bias, a.y, mean, rstd, a.s);
  else
    launch_norm_vec(a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? ICTC_OK : cuda_fail(e, "layer norm forward launch");
}

// Partial rows of dw and db that a backward of this shape may write, over both access
// widths (the workspace does not depend on the pointers).
constexpr int64_t kStreamRowParts = 64;

int64_t norm_parts(int64_t rows, int64_t width, size_t size, int device) {
  if (streams(width, true))
    return rows < kStreamRowParts ? rows : kStreamRowParts;
  const int a = plan_norm(rows, width, static_cast<int>(16 / size), device, true).grid;
  const int b = plan_norm(rows, width, 1, device, true).grid;
  return a > b ? a : b;
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
  const int vec = vector_width(sizeof(T), width, x_stride, g_stride, x, g, dx);
  a.p = plan_norm(rows, width, vec, current_device(), true);
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
  } else {
    launch_norm_vec(a);
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
