// Element types, activations and the column-sum reduction shared by the dense
// operators (layer norm, linear layer).
//
// Tensors are float32, bfloat16 or float16; every sum, statistic and activation is
// computed in float32 and rounded once when a tensor of the operand type is stored.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "common.cuh"

namespace ictc {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// N elements moved as one access of up to 16 bytes (more as several of them).
template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack {
  T v[N];
};

// exp(p) and 1 / p by the hardware's approximations (2 and 1 ulp, subnormals flushed),
// one instruction each; exp(p) = 2^(p log2 e), whose rounded argument costs 1.2 |p| ulp.
__device__ __forceinline__ float fast_exp(float p) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(p * 1.4426950408889634f));
  return r;
}

__device__ __forceinline__ float fast_reciprocal(float p) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(p));
  return r;
}

// 1 / (1 + exp(-p)), off by at most 2^-23 (the error of exp grows with |p|, but the
// sigmoid's slope falls faster), relative to the result by (4 + 1.2 |p|) 2^-23 where
// p < 0; exactly 0 where exp overflows.
__device__ __forceinline__ float sigmoid(float p) {
  return fast_reciprocal(1.f + fast_exp(-p));
}

// The standard normal distribution's upper tail at |p|, Q = (1 - erf(|p| / sqrt 2)) / 2, and
// exp(-p^2 / 2), without branches and with one exponential for both; erff took the
// epilogues half their time.  Q = exp(-p^2 / 2) t P(t) with t = 1 / (1 + 0.4 |p| / sqrt 2),
// the form of Abramowitz and Stegun 7.1.26; P is a weighted minimax fit of degree 7 made
// for this file (its relative error stays below 2^-23 up to |p| = 5.6, 2^-25 up to 2).  The
// published five coefficients leave 7.5e-8, twice what rounding does to gelu.
__device__ __forceinline__ float normal_tail(float p, float* density) {
  const float t = fast_reciprocal(fmaf(0.28284271f, fabsf(p), 1.f));
  const float e = fast_exp(-0.5f * (p * p));
  float q = fmaf(0.038026214f, t, -0.20159902f);
  q = fmaf(q, t, 0.35119181f);
  q = fmaf(q, t, -0.19723800f);
  q = fmaf(q, t, 0.21128423f);
  q = fmaf(q, t, 0.067113307f);
  q = fmaf(q, t, 0.11879680f);
  q = fmaf(q, t, 0.11242465f);
  *density = e;
  return q * t * e;
}

// act(p) and act'(p) for the activation codes of the C ABI.  ACT is the code, or
// kAnyActivation to take it from the argument (a branch that is uniform over a launch).
// gelu_tanh is written as p s(2 u), u = c (p + 0.044715 p^3): (1 + tanh u) / 2 = s(2 u).
constexpr int kAnyActivation = -1;

template <int ACT>
__device__ __forceinline__ float activate(float p, int any = ICTC_ACT_NONE) {
  const int code = ACT == kAnyActivation ? any : ACT;
  switch (code) {
    case ICTC_ACT_RELU:
      return p > 0.f ? p : (p != p ? p : 0.f);
    case ICTC_ACT_SILU:
      return p * sigmoid(p);
    case ICTC_ACT_GELU: {
      float e;
      const float q = normal_tail(p, &e);
      return p * (p >= 0.f ? 1.f - q : q);
    }
    case ICTC_ACT_GELU_TANH:
      return p * sigmoid(1.5957691216057308f * (p + 0.044715f * p * p * p));
    default:
      return p;
  }
}

template <int ACT>
__device__ __forceinline__ float activation_slope(float p, int any = ICTC_ACT_NONE) {
  const int code = ACT == kAnyActivation ? any : ACT;
  switch (code) {
    case ICTC_ACT_RELU:
      return p > 0.f ? 1.f : 0.f;
    case ICTC_ACT_SILU: {
      const float s = sigmoid(p);
      return s * (1.f + p * (1.f - s));
    }
    case ICTC_ACT_GELU: {
      float e;
      const float q = normal_tail(p, &e);
      return fmaf(p * 0.39894228040143268f, e, p >= 0.f ? 1.f - q : q);
    }
    case ICTC_ACT_GELU_TANH: {
      const float s = sigmoid(1.5957691216057308f * (p + 0.044715f * p * p * p));
      // s (1 - s) is 0 long before p^2 overflows, which would make a NaN of it
      const float p2 = fminf(p * p, 1e30f);
      return s + p * s * (1.f - s) * 1.5957691216057308f * fmaf(0.134145f, p2, 1.f);
    }
    default:
      return 1.f;
  }
}

inline size_t dtype_size(int dtype) { return dtype == ICTC_DTYPE_F32 ? 4 : 2; }

inline bool known_dtype(int dtype) {
  return dtype == ICTC_DTYPE_F32 || dtype == ICTC_DTYPE_BF16 || dtype == ICTC_DTYPE_F16;
}

inline size_t align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }

// out[c] = sum over p of partial[p * width + c], added in a fixed order: each of the
// 32 row lanes adds its rows p = lane, lane + 32, ... and the lanes' sums are added in
// lane order, so a result does not depend on scheduling.  Two column sums of one pass
// (weight and bias gradients) go in one launch through blockIdx.y.
constexpr int kColumnLanes = 32;

template <typename T>
static __global__ void __launch_bounds__(32 * kColumnLanes) column_total_kernel(
    const float* __restrict__ partial0, const float* __restrict__ partial1, T* __restrict__ out0,
    T* __restrict__ out1, int64_t parts, int64_t width) {
  __shared__ float sums[kColumnLanes][33];
  const float* partial = blockIdx.y ? partial1 : partial0;
  T* out = blockIdx.y ? out1 : out0;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x;
  float s = 0.f;
  if (c < width)
    for (int64_t p = threadIdx.y; p < parts; p += kColumnLanes) s += partial[p * width + c];
  sums[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < width) {
    float total = 0.f;
    for (int l = 0; l < kColumnLanes; ++l) total += sums[l][threadIdx.x];
    out[c] = from_float<T>(total);
  }
}

}  // namespace ictc
