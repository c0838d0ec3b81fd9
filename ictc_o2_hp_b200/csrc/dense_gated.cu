// The gated linear layer y = act(pg) pu, (pg | pu) = x W^T + b, and its gradients.
//
//   pg = x Wg^T + bg,  pu = x Wu^T + bu,  y = act(pg) pu
//   x [M, K], W = (Wg; Wu) [2 H, K] (gate rows first), b [2 H], pg, pu and y [M, H]
//   du = g act(pg),  dg = g pu act'(pg),  D = (dg | du) [M, 2 H]
//   dx = D W,  dW = D^T x,  db = sum_rows D
//
// With both halves of W in one tensor the backward's products are those of a linear layer of
// 2 H outputs without activation (dense_linear.cu), and so are the forward's sums here; the
// activation and the product of the halves are a pass over p = (pg | pu) in float32.
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "common.cuh"
#include "dense_types.cuh"

namespace ictc {
namespace {

int current_device() {
  int device = 0;
  return cudaGetDevice(&device) == cudaSuccess ? device : 0;
}

bool chunk_aligned(const void* p, int64_t ld, size_t size) {
  return aligned(p, 16) && (ld * static_cast<int64_t>(size)) % 16 == 0;
}

// Calls f with the activation code as a compile-time constant.
template <typename F>
void for_activation(int activation, const F& f) {
  switch (activation) {
    case ICTC_ACT_RELU: return f(std::integral_constant<int, ICTC_ACT_RELU>{});
    case ICTC_ACT_SILU: return f(std::integral_constant<int, ICTC_ACT_SILU>{});
    case ICTC_ACT_GELU: return f(std::integral_constant<int, ICTC_ACT_GELU>{});
    case ICTC_ACT_GELU_TANH: return f(std::integral_constant<int, ICTC_ACT_GELU_TANH>{});
    default: return f(std::integral_constant<int, ICTC_ACT_NONE>{});
  }
}

// --------------------------------------------------------------------- y = act(pg) pu
// One pass over p, bound by HBM.  V columns of each half a thread.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(256) gate_kernel(const float* __restrict__ p, T* __restrict__ y,
                                                   int64_t m, int64_t n) {
  const int64_t units = n / V, total = m * units;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += step) {
    const int64_t row = i / units, col = (i - row * units) * V;
    const Pack<float, V> g = *reinterpret_cast<const Pack<float, V>*>(p + row * 2 * n + col);
    const Pack<float, V> u = *reinterpret_cast<const Pack<float, V>*>(p + row * 2 * n + n + col);
    Pack<T, V> o;
#pragma unroll
    for (int j = 0; j < V; ++j) o.v[j] = from_float<T>(activate<ACT>(g.v[j]) * u.v[j]);
    *reinterpret_cast<Pack<T, V>*>(y + row * n + col) = o;
  }
}

// ------------------------------------------------------- D = (dg | du) and its column sums
// Bound by HBM.  A CTA owns a strip of columns of both halves and every gridDim.y-th block
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

int64_t aligned_pitch(int64_t width, size_t size) {
  const int64_t v = static_cast<int64_t>(16 / size);
  return ceil_div(width, v) * v;
}

int32_t layout_of(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t m, int64_t k,
                  size_t size) {
  int32_t flags = 0;
  if (chunk_aligned(x, ldx, size) && chunk_aligned(w, ldw, size)) flags |= ICTC_LINEAR_ALIGNED;
  if (aligned(x, 16) && (ldx == k || m <= 1)) flags |= ICTC_LINEAR_PACKED;
  return flags;
}

// Byte offsets of the workspace's parts, and its size.
struct GatedPlan {
  size_t p, y, d, columns, product, product_bytes, total;
};

constexpr int64_t kSlopeParts = 296;

// The forward's sums are a linear layer of 2 n outputs: p, and in 16-bit types the layer's
// own output, which nobody reads.
int plan_forward(int64_t m, int64_t n, int64_t k, int dtype, int32_t layout, bool keep, int device,
                 GatedPlan* b) {
  const size_t size = dtype_size(dtype);
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    const size_t here = at;
    at += align_up(bytes, 256);
    return here;
  };
  if (!keep) b->p = take(static_cast<size_t>(m) * 2 * n * sizeof(float));
  if (dtype != ICTC_DTYPE_F32) b->y = take(static_cast<size_t>(m) * 2 * n * size);
  size_t other;
  const int st = ictc_o2_linear_workspace(m, k, 2 * n, dtype, ICTC_ACT_NONE, layout, device,
                                          &b->product_bytes, &other);
  if (st != ICTC_OK) return st;
  b->product = take(b->product_bytes);
  b->total = at;
  return ICTC_OK;
}

int plan_backward(int64_t m, int64_t n, int64_t k, int dtype, int32_t layout, int device,
                  GatedPlan* b) {
  const size_t size = dtype_size(dtype);
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    const size_t here = at;
    at += align_up(bytes, 256);
    return here;
  };
  const int64_t pitch = aligned_pitch(2 * n, size);
  b->d = take(static_cast<size_t>(m) * pitch * size);
  b->columns = take(static_cast<size_t>(m < kSlopeParts ? m : kSlopeParts) * 2 * n * sizeof(float));
  const int32_t flags = layout & (pitch == 2 * n || m <= 1 ? ~0 : ~ICTC_LINEAR_PACKED);
  size_t other;
  const int st = ictc_o2_linear_workspace(m, k, 2 * n, dtype, ICTC_ACT_NONE, flags, device,
                                          &other, &b->product_bytes);
  if (st != ICTC_OK) return st;
  b->product = take(b->product_bytes);
  b->total = at;
  return ICTC_OK;
}

template <typename T>
int run_gate(const float* p, T* y, int64_t m, int64_t n, int activation, cudaStream_t stream) {
  const bool vec = n % 4 == 0 && aligned(y, 4 * sizeof(T)) && aligned(p, 16);
  const int64_t blocks = ceil_div(m * (vec ? n / 4 : n), 256);
  const int64_t cap = static_cast<int64_t>(sm_count(current_device())) * 8;
  const unsigned grid = static_cast<unsigned>(blocks < cap ? blocks : cap);
  for_activation(activation, [&](auto act) {
    if (vec) gate_kernel<T, 4, act.value><<<grid, 256, 0, stream>>>(p, y, m, n);
    else gate_kernel<T, 1, act.value><<<grid, 256, 0, stream>>>(p, y, m, n);
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

template <typename T>
int run_forward(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, void* y,
                float* preact, unsigned char* ws, const GatedPlan& plan, int64_t m, int64_t n,
                int64_t k, int dtype, int activation, cudaStream_t stream) {
  float* p = preact ? preact : reinterpret_cast<float*>(ws + plan.p);
  const bool wide = sizeof(T) == 4;
  const int st = ictc_o2_linear_forward(
      x, ldx, w, ldw, bias, nullptr, 0, wide ? static_cast<void*>(p) : ws + plan.y,
      wide ? nullptr : p, ws + plan.product, plan.product_bytes, m, k, 2 * n, dtype, ICTC_ACT_NONE,
      stream);
  return st != ICTC_OK ? st : run_gate<T>(p, static_cast<T*>(y), m, n, activation, stream);
}

template <typename T>
int run_backward(const void* x, int64_t ldx, const void* w, int64_t ldw, const float* p,
                 const void* g, int64_t ldg, void* dx, void* dw, void* db, unsigned char* ws,
                 const GatedPlan& plan, int64_t m, int64_t n, int64_t k, int dtype, int activation,
                 cudaStream_t stream) {
  T* d = dx || dw ? reinterpret_cast<T*>(ws + plan.d) : nullptr;
  const int64_t pitch = aligned_pitch(2 * n, sizeof(T));
  const int st = run_slope<T>(static_cast<const T*>(g), ldg, p, d, pitch,
                              reinterpret_cast<float*>(ws + plan.columns), static_cast<T*>(db), m,
                              n, activation, stream);
  if (st != ICTC_OK || !d) return st;
  return ictc_o2_linear_backward(x, ldx, w, ldw, nullptr, d, pitch, dx, dw, nullptr,
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
  st = plan_forward(rows, hidden, in, dtype, layout, keep != 0, device, &forward);
  if (st == ICTC_OK) st = plan_backward(rows, hidden, in, dtype, layout, device, &backward);
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
  if (x_stride < 0 || weight_stride < 0) return fail(ICTC_ERR_INVALID, "negative row stride");
  const int32_t layout =
      layout_of(x, x_stride, weight, weight_stride, rows, in, dtype_size(dtype));
  GatedPlan plan{};
  st = plan_forward(rows, hidden, in, dtype, layout, preact != nullptr, current_device(), &plan);
  if (st == ICTC_OK) st = check_workspace(workspace, workspace_bytes, plan.total);
  if (st != ICTC_OK) return st;
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define ICTC_GATED_FORWARD(T)                                                                  \
  return run_forward<T>(x, x_stride, weight, weight_stride, bias, y, preact, ws, plan, rows, \
                        hidden, in, dtype, activation, s)
  if (dtype == ICTC_DTYPE_F32) ICTC_GATED_FORWARD(float);
  if (dtype == ICTC_DTYPE_BF16) ICTC_GATED_FORWARD(__nv_bfloat16);
  ICTC_GATED_FORWARD(__half);
#undef ICTC_GATED_FORWARD
}

extern "C" int32_t ictc_o2_gated_linear_backward(
    const void* x, int64_t x_stride, const void* weight, int64_t weight_stride,
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
  if (!x || !weight || !grad_output || !preact) return fail(ICTC_ERR_INVALID, "null pointer");
  if (x_stride < 0 || weight_stride < 0 || grad_stride < 0)
    return fail(ICTC_ERR_INVALID, "negative row stride");
  const int32_t layout =
      layout_of(x, x_stride, weight, weight_stride, rows, in, dtype_size(dtype));
  GatedPlan plan{};
  st = plan_backward(rows, hidden, in, dtype, layout, current_device(), &plan);
  if (st == ICTC_OK) st = check_workspace(workspace, workspace_bytes, plan.total);
  if (st != ICTC_OK) return st;
  unsigned char* ws = static_cast<unsigned char*>(workspace);
#define ICTC_GATED_BACKWARD(T)                                                              \
  return run_backward<T>(x, x_stride, weight, weight_stride, preact, grad_output, grad_stride, \
                         grad_x, grad_weight, grad_bias, ws, plan, rows, hidden, in, dtype, \
                         activation, s)
  if (dtype == ICTC_DTYPE_F32) ICTC_GATED_BACKWARD(float);
  if (dtype == ICTC_DTYPE_BF16) ICTC_GATED_BACKWARD(__nv_bfloat16);
  ICTC_GATED_BACKWARD(__half);
#undef ICTC_GATED_BACKWARD
}
