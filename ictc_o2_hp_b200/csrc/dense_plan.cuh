// Host side shared by the linear layer and the gated one: how a product is cut into tiles and
// parts, and copies of operands whose rows lie off the 16-byte boundaries.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "common.cuh"
#include "dense_epilogue.cuh"
#include "dense_pair.cuh"
#include "dense_types.cuh"

namespace ictc {

constexpr int kBM = 128;  // rows of an output tile
constexpr int kBK = 64;   // K elements of a stage

inline int current_device() {
  int device = 0;
  return cudaGetDevice(&device) == cudaSuccess ? device : 0;
}

inline bool chunk_aligned(const void* p, int64_t ld, size_t size) {
  return aligned(p, 16) && (ld * static_cast<int64_t>(size)) % 16 == 0;
}

struct Split {
  int tiles_m, tiles_n, bn, chunks, splits, chunks_per_split;
  bool fits;  // tile counts fit the kernel's integers
};

// Parts of K that a 16-bit product needs for its sums' sake.  The tensor core truncates when
// it adds 16 products to an accumulator, always to the same side of a sum of one sign:
// measured, 2.3 2^-24 of the sum so far a step, 7e-5 of the whole after 16,384 elements and
// growing with their number, where rounding to float16 may be off by 2.4e-4.  Longer sums are
// taken in parts of at most 8,192 elements, joined in float32 (a limit of 8,192 for all would
// cost the training step of 16,384 x 4,096 x 4,096 44 us in 1,470).  float32 products move
// theirs out every 256 elements.
inline int64_t long_sum_parts(int64_t chunks) { return chunks <= 256 ? 1 : ceil_div(chunks, 128); }

// The K axis is split when the output has too few tiles to fill the SMs: at least four
// stages of K per split (the pipeline's depth), and no more splits than fill one wave unless
// long_sum_parts asks for them.
inline Split plan_product(int64_t m, int64_t n, int64_t k, bool f32, int device,
                          int most_columns = 128, int least_columns = 64) {
  Split s{};
  s.bn = (n <= 64 || most_columns == 64) && least_columns == 64 ? 64 : 128;
  const int64_t tm = ceil_div(m, kBM), tn = ceil_div(n, s.bn), chunks = ceil_div(k, kBK);
  s.fits = tm < (1ll << 31) && tn < (1ll << 31) && chunks < (1ll << 31);
  if (!s.fits) return s;
  s.tiles_m = static_cast<int>(tm);
  s.tiles_n = static_cast<int>(tn);
  s.chunks = static_cast<int>(chunks);
  const int64_t sms = sm_count(device);
  int64_t splits = tm * tn >= sms ? 1 : sms / (tm * tn);
  if (splits > chunks / 4) splits = chunks / 4;
  if (!f32 && splits < long_sum_parts(chunks)) splits = long_sum_parts(chunks);
  if (splits < 1) splits = 1;
  s.chunks_per_split = static_cast<int>(ceil_div(chunks, splits));
  s.splits = static_cast<int>(ceil_div(chunks, s.chunks_per_split));
  return s;
}

// ------------------------------------------------------------ 16-bit pairs: host side

struct PairPlan {
  bool ok;
  int bn, tiles_m, tiles_n, chunks, splits, chunks_per_split;
};

// Pairs take 16-bit products whose rows TMA can address, from one full 128 x 128 tile of
// work on.  BN is 256 unless 128-wide tiles leave the last wave of pairs fuller by more
// than they lose to the operand traffic in shared memory (192 instead of 128 bytes a
// cycle).  K is split as for the single-SM kernel, over pairs.
inline PairPlan plan_pair(int64_t m, int64_t n, int64_t k, int device) {
  PairPlan s{};
  if (m >= (1ll << 30) || n >= (1ll << 30) || k >= (1ll << 30)) return s;
  const int64_t pairs = sm_count(device) / 2, tm = ceil_div(m, kPairRows);
  const auto fill = [&](int64_t bn) {
    const int64_t tiles = tm * ceil_div(n, bn);
    const double waves = static_cast<double>(ceil_div(tiles, pairs));
    return static_cast<double>(m) * n / (waves * pairs * kPairRows * bn);
  };
  s.bn = n > 128 && fill(256) >= 0.65 * fill(128) ? 256 : 128;
  const int64_t tn = ceil_div(n, s.bn), chunks = ceil_div(k, 64);
  s.tiles_m = static_cast<int>(tm);
  s.tiles_n = static_cast<int>(tn);
  s.chunks = static_cast<int>(chunks);
  int64_t splits = tm * tn >= pairs ? 1 : pairs / (tm * tn);
  if (splits > chunks / 8) splits = chunks / 8;
  if (splits < long_sum_parts(chunks)) splits = long_sum_parts(chunks);
  if (splits < 1) splits = 1;
  s.chunks_per_split = static_cast<int>(ceil_div(chunks, splits));
  s.splits = static_cast<int>(ceil_div(chunks, s.chunks_per_split));
  s.ok = true;
  return s;
}

// The pair kernel needs a tile's worth of work to be worth its cluster start-up.
inline bool use_pair(int64_t m, int64_t n, int64_t k) {
  return static_cast<double>(m) * n * k >= static_cast<double>(1 << 21);
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

template <typename T>
bool vec_epilogue(const Epilogue& e, int64_t n) {
  return n % 4 == 0 && aligned(e.out, 4 * sizeof(T)) &&
         (!e.residual || (aligned(e.residual, 4 * sizeof(T)) && e.residual_stride % 4 == 0)) &&
         aligned(e.preact, 16);
}

// ------------------------------------------------------------- rows off the boundaries
// dst[r, :] = src[r, :] with a pitch of whole 16-byte blocks.
template <typename T>
static __global__ void __launch_bounds__(256)
    align_rows_kernel(const T* __restrict__ src, int64_t ld, T* __restrict__ dst, int64_t pitch,
                      int64_t rows, int64_t width) {
  constexpr int V = 16 / sizeof(T);
  const int64_t blocks = pitch / V;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < rows * blocks;
       i += step) {
    const int64_t r = i / blocks, c = (i - r * blocks) * V;
    Pack<T, V> pk;
#pragma unroll
    for (int j = 0; j < V; ++j) pk.v[j] = c + j < width ? src[r * ld + c + j] : T{};
    *reinterpret_cast<Pack<T, V>*>(dst + r * pitch + c) = pk;
  }
}

inline int64_t aligned_pitch(int64_t width, size_t size, int64_t unit = 16) {
  const int64_t v = unit / static_cast<int64_t>(size);
  return ceil_div(width, v) * v;
}

// Element-by-element loads of unaligned rows cost the products several times their time;
// copying the operand first costs one pass over it and a launch.
inline bool worth_aligning(int64_t m, int64_t n, int64_t k) {
  return static_cast<double>(m) * n * k >= static_cast<double>(1 << 26);
}

// An operand with aligned rows: itself, or its copy in `space`, whose rows are whole blocks of
// `unit` bytes.
template <typename T>
static int align_operand(const T** p, int64_t* ld, int64_t rows, int64_t width,
                         unsigned char* space, cudaStream_t stream, int64_t unit = 16) {
  if (chunk_aligned(*p, *ld, sizeof(T))) return ICTC_OK;
  const int64_t pitch = aligned_pitch(width, sizeof(T), unit);
  T* to = reinterpret_cast<T*>(space);
  const int64_t blocks = ceil_div(rows * pitch * static_cast<int64_t>(sizeof(T)), 256 * 16);
  const int64_t cap = static_cast<int64_t>(sm_count(current_device())) * 8;
  align_rows_kernel<T><<<static_cast<unsigned>(blocks < cap ? blocks : cap), 256, 0, stream>>>(
      *p, *ld, to, pitch, rows, width);
  *p = to;
  *ld = pitch;
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? ICTC_OK : cuda_fail(e, "linear operand copy launch");
}

}  // namespace ictc
