// The linear layer y = act(x W^T + b) + r and its gradients.
//
//   p = x W^T + b,  y = act(p) + r           x [M, K], W [N, K], p and y [M, N]
//   d = g act'(p),  dx = d W,  dW = d^T x,  db = sum_rows d,  dr = g
//
// Every product runs on the tensor cores with float32 accumulators in TMEM.  16-bit
// operands enter as they are.  A float32 value is cut exactly into three bf16 parts of
// eight significant bits each (x = x1 + x2 + x3, by truncation), and six of the nine
// partial products are summed:
//   a b ~ a1 b1 + (a1 b2 + a2 b1 + a2 b2 + a1 b3 + a3 b1)
// The three left out are each below 2^-22 of |a b|, and mostly far below.  The tensor core
// truncates when it adds to an accumulator, so the large first term and the small others
// have accumulators of their own, and both are moved into registers and added there,
// rounded to nearest, every 256 elements of K.  Errors against 64 bits in the 2-norm, beside
// those of PyTorch's float32 operations: 1.0e-7 and 0.7e-7 for 37 x 8 x 64, 4e-7 and 7e-7 for
// a training step of 65,536 x 128 x 512, 4e-7 and 2e-6 for 1,048,576 x 64 x 64.  An
// infinity or NaN in an operand is its own leading part, and decides an element through
// the sum of a1 b1 alone (join_parts).  Two things are given up for that: an infinity that
// meets a subnormal below 2^-133, whose leading part is zero, gives NaN; and a signalling
// NaN with nothing in its upper seven bits of payload, which no arithmetic produces, counts
// as an infinity.
//
// Which kernel a product takes:
//   up to 4 rows, aligned (forward)             FMAs, W read once (few_rows_kernel)
//   a dimension of at most 8                    FMAs, the large operand read once, in any
//                                               layout (dense_thin.cuh; thin_form and
//                                               plan_linear have the exceptions)
//   up to 64 inputs and outputs, contiguous     one kernel per direction (dense_narrow.cuh)
//   16-bit, aligned rows                        SM pairs fed by TMA (dense_pair.cuh)
//   float32, aligned rows                       cut on the way in (dense_cut.cuh)
//   anything else: small or unaligned           register-staged operands (product_kernel);
//                                               large ones are copied to aligned rows first
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "common.cuh"
#include "dense_cut.cuh"
#include "dense_epilogue.cuh"
#include "dense_narrow.cuh"
#include "dense_pair.cuh"
#include "dense_plan.cuh"
#include "dense_thin.cuh"
#include "dense_types.cuh"
#include "tcgen05.cuh"
#include "tmap.cuh"

namespace ictc {
namespace {

constexpr int kEpilogueWarps = 8;  // warps 0-7
constexpr int kProducerWarps = 8;  // warps 8-15
constexpr int kMmaWarp = kEpilogueWarps;  // the producer warp whose lane 0 issues the MMAs
constexpr int kProductThreads = (kEpilogueWarps + kProducerWarps) * 32;
constexpr int kGroupChunks = 4;    // float32: K stages between moves into registers

template <typename T>
constexpr int kPieces = sizeof(T) == 4 ? 3 : 1;

template <typename T, int BN>
constexpr int kStageBytes = kPieces<T> * (kBM + BN) * 128;

template <typename T, int BN>
constexpr int kStages = sizeof(T) == 4 ? 2 : 4;

constexpr int kStagingBytes = kEpilogueWarps * 4096;

template <typename T, int BN>
constexpr size_t kProductSmem = 1024 + kStages<T, BN> * kStageBytes<T, BN> + kStagingBytes + 128;

// ------------------------------------------------------------------ operand loading
// 256 producer threads bring one [ROWS x 64] operand chunk: CH pieces of eight
// consecutive elements each.  Elements outside the operand read as zero.

template <typename T, int ROWS>
struct Held {
  Pack<T, 8> v[ROWS / 32];
};

template <typename T, bool MN, int ROWS>
__device__ __forceinline__ void chunk_place(int tid, int i, int* row, int* c) {
  // K-major: 8 chunks per row; MN-major: ROWS / 8 chunks per k
  constexpr int kPerRow = MN ? ROWS / 8 : 8;
  *c = tid % kPerRow;
  *row = tid / kPerRow + i * (256 / kPerRow);
}

template <typename T, bool MN, int ROWS>
__device__ __forceinline__ void load_operand(const T* base, int64_t ld, int64_t mn0,
                                             int64_t extent, int64_t k0, int64_t k_end, bool vec,
                                             int tid, Held<T, ROWS>& h) {
  int row0, c;
  chunk_place<T, MN, ROWS>(tid, 0, &row0, &c);
  constexpr int kRowStep = 256 / (MN ? ROWS / 8 : 8);
  const int64_t inner = (MN ? mn0 : k0) + c * 8;  // first contiguous index
  const int64_t inner_left = (MN ? extent : k_end) - inner;
  const int left = inner_left < 8 ? (inner_left < 0 ? 0 : static_cast<int>(inner_left)) : 8;
  const int64_t outer_left = (MN ? k_end - k0 : extent - mn0) - row0;  // along the stride
  const int rows_left = outer_left < ROWS ? static_cast<int>(outer_left) : ROWS;
  const T* src = base + ((MN ? k0 : mn0) + row0) * ld + inner;
  const int64_t step = kRowStep * ld;
#pragma unroll
  for (int i = 0; i < ROWS / 32; ++i, src += step) {
    const bool in = i * kRowStep < rows_left;
    if (in && vec && left == 8) {
      if constexpr (sizeof(T) == 4) {
        const float4 lo = __ldg(reinterpret_cast<const float4*>(src));
        const float4 hi = __ldg(reinterpret_cast<const float4*>(src) + 1);
        h.v[i].v[0] = lo.x; h.v[i].v[1] = lo.y; h.v[i].v[2] = lo.z; h.v[i].v[3] = lo.w;
        h.v[i].v[4] = hi.x; h.v[i].v[5] = hi.y; h.v[i].v[6] = hi.z; h.v[i].v[7] = hi.w;
      } else {
        *reinterpret_cast<uint4*>(&h.v[i]) = __ldg(reinterpret_cast<const uint4*>(src));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        h.v[i].v[j] = in && j < left ? src[j] : T{};
    }
  }
}

template <typename T, bool MN, int ROWS>
__device__ __forceinline__ void store_operand(unsigned char* dst, int tid,
                                              const Held<T, ROWS>& h) {
#pragma unroll
  for (int i = 0; i < ROWS / 32; ++i) {
    int row, c;
    chunk_place<T, MN, ROWS>(tid, i, &row, &c);
    // MN-major tiles wider than 64 are blocks of [64 k rows][128 bytes]
    const uint32_t at = MN ? (c >> 3) * (kBK * 128) + swizzled(row, c & 7) : swizzled(row, c);
    if constexpr (sizeof(T) == 4) {
      uint32_t part[4][3];
#pragma unroll
      for (int j = 0; j < 4; ++j) cut_pair(h.v[i].v[2 * j], h.v[i].v[2 * j + 1], part[j]);
#pragma unroll
      for (int q = 0; q < 3; ++q)
        *reinterpret_cast<uint4*>(dst + q * ROWS * 128 + at) =
            make_uint4(part[0][q], part[1][q], part[2][q], part[3][q]);
    } else {
      *reinterpret_cast<uint4*>(dst + at) = *reinterpret_cast<const uint4*>(&h.v[i]);
    }
  }
}

// One thread: the products of a stage, `steps` K steps of 16.  `add` false starts new sums.
template <typename T, bool A_MN, bool B_MN, int BN>
__device__ __forceinline__ void issue_stage(uint32_t sa, uint32_t d, int steps, bool add) {
  constexpr int P = kPieces<T>;
  constexpr uint32_t kDesc =
      mma_descriptor(!std::is_same_v<T, __half>, A_MN, B_MN, kBM, BN);
  // a step's 16 elements along K: 32 bytes of a K-major row, 16 rows MN-major; piece
  // bytes and steps are multiples of 16, the unit of the descriptor's address field
  constexpr uint64_t kA = A_MN ? 128 : 2, kB = B_MN ? 128 : 2;
  constexpr uint64_t kPa = kBM * 8, kPb = BN * 8;
  uint64_t a = matrix_descriptor(sa, kBK * 128, 1024);
  uint64_t b = matrix_descriptor(sa + P * kBM * 128, kBK * 128, 1024);
#pragma unroll 1
  for (int k = 0; k < steps; ++k, a += kA, b += kB) {
    mma_f16(d, a, b, kDesc, add);
    if constexpr (P == 3) {
      mma_f16(d + BN, a + 2 * kPa, b, kDesc, add);
      mma_f16(d + BN, a, b + 2 * kPb, kDesc, true);
      mma_f16(d + BN, a + kPa, b + kPb, kDesc, true);
      mma_f16(d + BN, a + kPa, b, kDesc, true);
      mma_f16(d + BN, a, b + kPb, kDesc, true);
    }
    add = true;
  }
}

// ---------------------------------------------------------------------- the product
// For operands that TMA cannot address (and 16-bit products below a tile of work).
// One persistent CTA per SM, warps specialised: 8 producer warps load operand chunks
// into registers, cut float32 values and store the swizzled tiles; one of their threads
// issues the MMAs of a stage; 8 epilogue warps move finished accumulators out of TMEM, which holds
// two sets, so a tile's epilogue overlaps the next tile's products.
template <typename T, bool A_MN, bool B_MN, int BN, int ACT>
__global__ void __launch_bounds__(kProductThreads, 1) product_kernel(const __grid_constant__ ProductArgs p) {
  constexpr int P = kPieces<T>;
  constexpr int S = kStages<T, BN>;
  constexpr uint32_t kABytes = kBM * 128;
  constexpr uint32_t kSet = (P == 3 ? 2 : 1) * BN;  // TMEM columns of one accumulator set
  constexpr uint32_t kColumns = 2 * kSet;
  extern __shared__ unsigned char raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t{1023});
  unsigned char* staging = smem + S * kStageBytes<T, BN>;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + kStagingBytes);
  uint64_t* empty = full + S;
  uint64_t* done = empty + S;   // accumulator set ready for the epilogue
  uint64_t* room = done + 2;    // accumulator set free for the MMAs
  uint64_t* drain = room + 2;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(drain + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], kProducerWarps);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&done[s], 1);
      mbar_init(&room[s], kEpilogueWarps);
    }
    mbar_init(drain, 1);
    fence_mbarrier_init();
  }
  if (warp == kMmaWarp) tmem_alloc(tmem_at, kColumns);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = *tmem_at;
  const int64_t total = static_cast<int64_t>(p.tiles_m) * p.tiles_n * p.splits;

  if (warp >= kEpilogueWarps) {
    // ---- producers; lane 0 of the first also issues each stage's MMAs.  (A warp of its
    // own for them would cost every thread 32 of its 128 registers: registers are given
    // out to four warps at a time.)
    const int tid = threadIdx.x - kEpilogueWarps * 32;
    const T* a = static_cast<const T*>(p.a);
    const T* b = static_cast<const T*>(p.b);
    int64_t t = blockIdx.x;
    bool ok = true;
    uint32_t it = 0, set = 0, in_group = 0;
    Held<T, kBM> ha;
    Held<T, BN> hb;
    TilePos pos = tile_at<kBM>(p, t, BN);
    int c = pos.c0;
    load_operand<T, A_MN, kBM>(a, p.lda, pos.m0, p.m, static_cast<int64_t>(c) * kBK, p.k, p.vec_a,
                               tid, ha);
    for (bool more = true; more; ++it) {
      load_operand<T, B_MN, BN>(b, p.ldb, pos.n0, p.n, static_cast<int64_t>(c) * kBK, p.k,
                                p.vec_b, tid, hb);
      const int s = it % S;
      ok = mbar_wait_warp(&empty[s], ((it / S) & 1) ^ 1, kCodeProducer);
      if (!ok) break;
      unsigned char* stage = smem + s * kStageBytes<T, BN>;
      store_operand<T, A_MN, kBM>(stage, tid, ha);
      // the next chunk's A is in flight while this chunk's B is cut and stored
      const int64_t left = p.k - static_cast<int64_t>(c) * kBK;
      const bool last = ++c == pos.c1;
      if (last) {
        t += gridDim.x;
        more = t < total;
        if (more) {
          pos = tile_at<kBM>(p, t, BN);
          c = pos.c0;
        }
      }
      if (more)
        load_operand<T, A_MN, kBM>(a, p.lda, pos.m0, p.m, static_cast<int64_t>(c) * kBK, p.k,
                                   p.vec_a, tid, ha);
      store_operand<T, B_MN, BN>(stage + P * kABytes, tid, hb);
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[s]);
      if (warp == kMmaWarp) {
        const bool close = last || (P == 3 && in_group == kGroupChunks - 1);
        if (lane == 0) {
          if (in_group == 0) ok = mbar_wait_idle(&room[set & 1], ((set >> 1) & 1) ^ 1, kCodeMma);
          if (ok) ok = mbar_wait_idle(&full[s], (it / S) & 1, kCodeMma);
          if (ok) {
            tcgen05_fence_after();
            issue_stage<T, A_MN, B_MN, BN>(smem_addr(stage), tmem + (set & 1) * kSet,
                                           left < kBK ? static_cast<int>((left + 15) / 16)
                                                      : kBK / 16,
                                           in_group > 0);
            mma_commit(&empty[s]);
            if (close) mma_commit(&done[set & 1]);
          }
        }
        ok = __shfl_sync(0xffffffffu, static_cast<int>(ok), 0) != 0;
        if (!ok) break;
        in_group = close ? 0 : in_group + 1;
        set += close ? 1 : 0;
      }
    }
    if (!ok && warp == kMmaWarp) {
      // let the MMAs in flight finish before TMEM and the stages go away
      if (lane == 0) {
        mma_commit(drain);
        mbar_wait(drain, 0, kCodeDrain, kDrainLimitNs);
      }
      __syncwarp();
    }
  } else {
    // ---- epilogue: warp w holds TMEM lanes 32 (w % 4) .. + 31, half w / 4 of the columns
    constexpr int kHalf = BN / 2;
    const int quad = warp & 3, half = warp >> 2;
    float4* mine = reinterpret_cast<float4*>(staging + warp * 4096);
    bool ok = true;
    uint32_t set = 0;
    for (int64_t t = blockIdx.x; ok && t < total; t += gridDim.x) {
      const TilePos pos = tile_at<kBM>(p, t, BN);
      const int64_t row0 = pos.m0 + quad * 32;
      ResidualBlock<T> res;
      load_residual(p, row0, pos.n0 + half * kHalf, lane, res);
      float acc[kHalf];
      const int groups = P == 3 ? (pos.c1 - pos.c0 + kGroupChunks - 1) / kGroupChunks : 1;
      for (int gi = 0; gi < groups; ++gi, ++set) {
        ok = mbar_wait_warp(&done[set & 1], (set >> 1) & 1, kCodeEpilogue);
        if (!ok) break;
        tcgen05_fence_after();
        const uint32_t at =
            tmem + (set & 1) * kSet + (static_cast<uint32_t>(quad * 32) << 16) + half * kHalf;
#pragma unroll
        for (int j = 0; j < kHalf; j += 16) {
          float v[16];
          tmem_load16(at + j, v);
          if constexpr (P == 3) {
            float y[16];
            tmem_load16(at + BN + j, y);
            tmem_load_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = join_parts(v[i], y[i]);
          } else {
            tmem_load_wait();
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[j + i] = gi == 0 ? v[i] : acc[j + i] + v[i];
        }
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&room[set & 1]);
      }
      if (!ok) break;
#pragma unroll
      for (int cb = 0; cb < kHalf / 32; ++cb) {
        const int64_t col0 = pos.n0 + half * kHalf + cb * 32;
        write_block<T, ACT>(p, pos.split, acc + cb * 32, mine, row0, col0, lane, res);
        if (cb + 1 < kHalf / 32) load_residual(p, row0, col0 + 32, lane, res);
      }
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tcgen05_fence_after();
    tmem_free(tmem, kColumns);
  }
}

// out = epilogue(sum of the splits' partial products), the splits added in order.  Rows of
// whole quads lie behind one another: their quads are numbered through, four to a thread so
// that their loads are in flight together.
template <typename T>
__global__ void __launch_bounds__(256) join_splits_kernel(const Epilogue e, int64_t m, int64_t n,
                                                          int splits) {
  constexpr int kAhead = 4;
  const int64_t quads = (n + 3) / 4, total = m * quads;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
  int64_t q = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (e.vec) {
    const float4* parts = reinterpret_cast<const float4*>(e.partial);
    const bool placed = e.bias || e.residual;
    for (; q < total; q += kAhead * step) {
      float4 sum[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (q + u * step < total) sum[u] = parts[q + u * step];
      for (int s = 1; s < splits; ++s) {
        const float4* part = parts + s * total + q;
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
          if (q + u * step < total) {
            const float4 f = part[u * step];
            sum[u].x += f.x; sum[u].y += f.y; sum[u].z += f.z; sum[u].w += f.w;
          }
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int64_t at = q + u * step;
        if (at >= total) break;
        float v[4] = {sum[u].x, sum[u].y, sum[u].z, sum[u].w}, bias[4] = {0.f, 0.f, 0.f, 0.f};
        Pack<T, 4> r{};
        if (placed) {
          const int64_t row = at / quads, col = (at - row * quads) * 4;
          load_bias4<T>(e, col, n, bias);
          if (e.residual) r = residual4<T>(e, row, col);
        }
        finish4<T, kAnyActivation>(e, at * 4, v, bias, r);
      }
    }
    return;
  }
  for (; q < total; q += step) {
    const int64_t row = q / quads, col = (q - row * quads) * 4;
    const float* at = e.partial + row * n + col;
    for (int j = 0; j < 4 && col + j < n; ++j) {
      float v = 0.f;
      for (int s = 0; s < splits; ++s) v += at[s * m * n + j];
      finish1<T, kAnyActivation>(e, row, col + j, n, v,
                                 e.bias ? to_float(static_cast<const T*>(e.bias)[col + j]) : 0.f);
    }
  }
}

// ---------------------------------------------------------------- few rows: no tiles
// Up to four rows: W is read once and the products run on the FMA pipes (bf16 1 x 4,096 x
// 4,096: 7.0 us, 4.8 TB/s).
// W_ warps share one output column, each a part of K; a lane reads V consecutive
// elements, the warps' sums are added in warp order.
constexpr int kRowThreads = 256;

template <typename T, int ROWS, int V>
__global__ void __launch_bounds__(kRowThreads) few_rows_kernel(
    const T* __restrict__ x, int64_t ldx, const T* __restrict__ w, int64_t ldw, int64_t rows,
    int64_t n, int64_t k, int share, const Epilogue e) {
  __shared__ float sums[kRowThreads / 32][ROWS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_cta = (kRowThreads / 32) / share;  // columns per CTA and round
  const int part = warp % share;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * per_cta; base < n;
       base += static_cast<int64_t>(gridDim.x) * per_cta) {
    const int64_t col = base + warp / share;
    float acc[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) acc[r] = 0.f;
    if (col < n) {
      const T* wr = w + col * ldw;
#pragma unroll 4
      for (int64_t c = (part * 32 + lane) * V; c < k; c += share * 32 * V) {
        const Pack<T, V> pw = *reinterpret_cast<const Pack<T, V>*>(wr + c);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          if (r >= rows) break;
          const Pack<T, V> px = *reinterpret_cast<const Pack<T, V>*>(x + r * ldx + c);
#pragma unroll
          for (int j = 0; j < V; ++j) acc[r] = fmaf(to_float(px.v[j]), to_float(pw.v[j]), acc[r]);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], o);
    if (share > 1) {
      if (lane == 0)
#pragma unroll
        for (int r = 0; r < ROWS; ++r) sums[warp][r] = acc[r];
      __syncthreads();
      if (part == 0)
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          acc[r] = 0.f;
          for (int q = 0; q < share; ++q) acc[r] += sums[warp + q][r];
        }
      __syncthreads();
    }
    if (part == 0 && lane == 0 && col < n) {
      const float bias = e.bias ? to_float(static_cast<const T*>(e.bias)[col]) : 0.f;
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        if (r >= rows) break;
        const float v = acc[r] + bias;
        if (e.preact) e.preact[r * n + col] = v;
        float y = activate<kAnyActivation>(v, e.activation);
        if (e.residual)
          y += to_float(static_cast<const T*>(e.residual)[r * e.residual_stride + col]);
        static_cast<T*>(e.out)[r * n + col] = from_float<T>(y);
      }
    }
  }
}

// ------------------------------------------------------- d = g act'(p) and sums of d
// Bound by HBM (bf16 16,384 x 4,096: 120 us, 4.5 TB/s; float32 65,536 x 512: 68 us, 5.9 TB/s).
// A CTA owns a strip of columns and every gridDim.y-th block of rows; each
// thread keeps its columns' sums in registers, and the CTA's partial row of db is joined
// over its row lanes in order.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(256) slope_kernel(const T* __restrict__ g, int64_t ldg,
                                                    const float* __restrict__ preact,
                                                    T* __restrict__ d, int64_t ldd,
                                                    float* __restrict__ partial,
                                                    T* __restrict__ db, int64_t m, int64_t n,
                                                    int lanes) {
  __shared__ float sums[256 * V];
  const int tx = threadIdx.x % lanes, ty = threadIdx.x / lanes, rows = 256 / lanes;
  const int64_t col = (static_cast<int64_t>(blockIdx.x) * lanes + tx) * V;
  float acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.f;
  if (col < n) {
    constexpr int kAhead = 4;  // rows whose loads go out together, ahead of any store
    const int64_t step = static_cast<int64_t>(gridDim.y) * rows;
    for (int64_t r0 = static_cast<int64_t>(blockIdx.y) * rows + ty; r0 < m; r0 += kAhead * step) {
      Pack<T, V> pg[kAhead];
      Pack<float, V> pp[kAhead];
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        const int64_t r = r0 + q * step;
        pg[q] = Pack<T, V>{};
        if (r < m) {
          pg[q] = *reinterpret_cast<const Pack<T, V>*>(g + r * ldg + col);
          if constexpr (ACT != ICTC_ACT_NONE) {
            pp[q] = *reinterpret_cast<const Pack<float, V>*>(preact + r * n + col);
          }
        }
      }
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        const int64_t r = r0 + q * step;
        if (r >= m) break;
        Pack<T, V> o;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float v = to_float(pg[q].v[j]);
          if constexpr (ACT != ICTC_ACT_NONE) v *= activation_slope<ACT>(pp[q].v[j]);
          acc[j] += v;
          o.v[j] = from_float<T>(v);
        }
        if constexpr (ACT != ICTC_ACT_NONE) *reinterpret_cast<Pack<T, V>*>(d + r * ldd + col) = o;
      }
    }
  }
  if (partial == nullptr) return;
#pragma unroll
  for (int j = 0; j < V; ++j) sums[(ty * lanes + tx) * V + j] = acc[j];
  __syncthreads();
  for (int c = threadIdx.x; c < lanes * V; c += 256) {
    const int64_t at = static_cast<int64_t>(blockIdx.x) * lanes * V + c;
    if (at >= n) break;
    float total = 0.f;
    for (int q = 0; q < rows; ++q) total += sums[q * lanes * V + c];
    if (db != nullptr) db[at] = from_float<T>(total);
    else partial[blockIdx.y * n + at] = total;
  }
}

// ----------------------------------------------------------------------- host side


// Bytes of partial products, whichever kernel a call's pointers let it take.
size_t split_bytes(int64_t m, int64_t n, int64_t k, int dtype, int device) {
  int64_t splits = plan_product(m, n, k, dtype == ICTC_DTYPE_F32, device).splits;
  if (dtype != ICTC_DTYPE_F32) {
    const int64_t q = plan_pair(m, n, k, device).splits;
    if (q > splits) splits = q;
  }
  return splits > 1 ? static_cast<size_t>(splits) * m * n * sizeof(float) : 0;
}

// The epilogue that a launch needs: gradients and partial sums have no activation.
template <bool FORWARD, typename F>
void for_epilogue(const ProductArgs& p, const F& f) {
  if constexpr (FORWARD)
    for_activation(p.e.partial ? ICTC_ACT_NONE : p.e.activation, f);
  else
    f(std::integral_constant<int, ICTC_ACT_NONE>{});
}

template <typename T, bool A_MN, bool B_MN, int BN>
int launch_pair(const OperandMaps& maps, const ProductArgs& p, int device, cudaStream_t stream) {
  const int64_t total = static_cast<int64_t>(p.tiles_m) * p.tiles_n * p.splits;
  const int64_t pairs = sm_count(device) / 2;
  const unsigned grid = static_cast<unsigned>(2 * (total < pairs ? total : pairs));
  int st = ICTC_OK;
  for_epilogue<!A_MN && !B_MN>(p, [&](auto act) {
    const auto kernel = pair_product_kernel<T, A_MN, B_MN, BN, act.value>;
    st = allow_smem(reinterpret_cast<const void*>(kernel), kPairSmem<BN>);
    if (st == ICTC_OK) kernel<<<grid, kPairThreads, kPairSmem<BN>, stream>>>(maps, p);
  });
  if (st != ICTC_OK) return st;
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? ICTC_OK : cuda_fail(e, "linear pair product launch");
}

template <bool A_MN, bool B_MN, int BN>
int launch_cut(const OperandMaps& maps, const ProductArgs& p, int device, cudaStream_t stream) {
  const int64_t total = static_cast<int64_t>(p.tiles_m) * p.tiles_n * p.splits;
  const int64_t sms = sm_count(device);
  const unsigned grid = static_cast<unsigned>(total < sms ? total : sms);
  int st = ICTC_OK;
  for_epilogue<!A_MN && !B_MN>(p, [&](auto act) {
    const auto kernel = cut_product_kernel<A_MN, B_MN, BN, act.value>;
    if (!cut_shares_fit<A_MN, B_MN, BN, act.value>()) {
      st = fail(ICTC_ERR_UNSUPPORTED,
                "float32 product: built with fewer than %d registers a thread",
                kCutLaunchRegisters);
      return;
    }
    st = allow_smem(reinterpret_cast<const void*>(kernel), kCutSmem<BN>);
    if (st == ICTC_OK) kernel<<<grid, kCutThreads, kCutSmem<BN>, stream>>>(maps, p);
  });
  if (st != ICTC_OK) return st;
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? ICTC_OK : cuda_fail(e, "linear float32 product launch");
}

template <typename T, bool A_MN, bool B_MN, int BN>
int launch_product(const ProductArgs& p, int device, cudaStream_t stream) {
  const int64_t total = static_cast<int64_t>(p.tiles_m) * p.tiles_n * p.splits;
  const int64_t sms = sm_count(device);
  const unsigned grid = static_cast<unsigned>(total < sms ? total : sms);
  int st = ICTC_OK;
  const auto launch = [&](auto act) {
    const auto kernel = product_kernel<T, A_MN, B_MN, BN, act.value>;
    st = allow_smem(reinterpret_cast<const void*>(kernel), kProductSmem<T, BN>);
    if (st == ICTC_OK) kernel<<<grid, kProductThreads, kProductSmem<T, BN>, stream>>>(p);
  };
  // products come here only when small or unaligned: one kernel for every activation
  launch(std::integral_constant<int, kAnyActivation>{});
  if (st != ICTC_OK) return st;
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? ICTC_OK : cuda_fail(e, "linear product launch");
}

// --------------------------------------------------------------- thin forms: host side

enum class Thin { none, dot, dot_swapped, outer, gram, gram_swapped };

int thin_columns(int64_t count) {
  return count <= 2 ? static_cast<int>(count) : count <= 4 ? 4 : kThin;
}

// The staged operand fits, and there are rows enough to fill the SMs without splitting the
// sum (or it is short).
bool dot_fits(int64_t rows, int64_t len, int64_t count) {
  return len <= static_cast<int64_t>(kThinBytes / sizeof(float)) / thin_columns(count) - 3 &&
         (rows >= 1024 || len <= 8192);
}

// Whether a large 16-bit product goes to the SM pairs all the same: with TMA (`tiles`) their
// mostly empty tiles still read it at up to 4.6 TB/s, where from three (dot) or five (outer,
// gram) numbers a value on the FMAs and conversions take longer.  bf16 16,384 x 4,096 x 8
// forward 29 us (dot 83), x 1 30 (26); 65,536 x 1,024 x 4 forward 30 (dot 38), dx 77 (outer 65),
// dW 55 (gram 54); 8 x 4,096 x 16,384 dx 47 (gram 79), dW 77 (outer 89).  float32 tiles do not
// (16,384 x 4,096 x 8 forward 111 us, dot 61).
bool pairs_read_faster(bool tiles, int64_t one, int64_t two, int64_t count, int64_t most) {
  return tiles && count > most && one > kNarrow && two > kNarrow && one * two >= (1 << 21);
}

// The form of a product with a dimension of at most kThin.  A few rows over a weight whose
// rows run along the sum (the forward's) are decided by the caller.
Thin thin_form(bool a_mn, bool b_mn, int64_t m, int64_t n, int64_t k, bool tiles) {
  if (k <= kThin) return pairs_read_faster(tiles, m, n, k, 4) ? Thin::none : Thin::outer;
  if (n <= kThin && a_mn)
    return pairs_read_faster(tiles, m, k, n, 4) ? Thin::none : Thin::gram_swapped;
  if (n <= kThin && dot_fits(m, k, n))
    return pairs_read_faster(tiles, m, k, n, 2) ? Thin::none : Thin::dot;
  if (m <= kThin && b_mn) return pairs_read_faster(tiles, n, k, m, 4) ? Thin::none : Thin::gram;
  return Thin::none;
}

struct StripPlan {
  int lanes;
  unsigned blocks_x, blocks_y;
};

// Strips of 32 lanes of `vec` (or, strided, four) columns, and as many blocks of rows as fill
// the SMs, each thread's at least four rows (the loads that it has in flight).
StripPlan plan_strips(int64_t rows, int64_t width, int vec, int device) {
  StripPlan s{};
  const int64_t units = ceil_div(width, vec > 1 ? vec : kStrided);
  s.lanes = 1;
  while (s.lanes < 32 && s.lanes < units) s.lanes *= 2;
  s.blocks_x = static_cast<unsigned>(ceil_div(units, s.lanes));
  const int64_t most = ceil_div(rows, 4 * (kStripThreads / s.lanes));
  int64_t y = ceil_div(static_cast<int64_t>(sm_count(device)) * 8, s.blocks_x);
  if (y > 296) y = 296;
  if (y > most) y = most;
  s.blocks_y = static_cast<unsigned>(y < 1 ? 1 : y);
  return s;
}

// Bytes of a gram form's partial sums, whichever access width the pointers allow.
size_t gram_bytes(int64_t rows, int64_t width, int64_t count, size_t size, int device) {
  size_t parts = 1;
  for (const int vec : {static_cast<int>(16 / size), 1}) {
    const size_t y = plan_strips(rows, width, vec, device).blocks_y;
    if (y > parts) parts = y;
  }
  return parts * static_cast<size_t>(width) * count * sizeof(float);
}

// Workspace of a product, whichever kernel it takes.
size_t product_bytes(bool a_mn, bool b_mn, int64_t m, int64_t n, int64_t k, int dtype,
                     int device) {
  const size_t size = dtype_size(dtype), tiles = split_bytes(m, n, k, dtype, device);
  size_t thin = 0;
  const Thin form = thin_form(a_mn, b_mn, m, n, k, false);
  if (form == Thin::gram) thin = gram_bytes(k, n, m, size, device);
  if (form == Thin::gram_swapped) thin = gram_bytes(k, m, n, size, device);
  return tiles > thin ? tiles : thin;
}

// Calls f with the small dimension as a compile-time constant.
template <typename F>
void for_thin(int count, const F& f) {
  switch (count) {
    case 1: return f(std::integral_constant<int, 1>{});
    case 2: return f(std::integral_constant<int, 2>{});
    case 3: return f(std::integral_constant<int, 3>{});
    case 4: return f(std::integral_constant<int, 4>{});
    case 5: return f(std::integral_constant<int, 5>{});
    case 6: return f(std::integral_constant<int, 6>{});
    case 7: return f(std::integral_constant<int, 7>{});
    default: return f(std::integral_constant<int, kThin>{});
  }
}

// Rows that a group of lanes holds at a time: several share every read of the staged operand,
// as long as that leaves work for all warps of the SMs.
template <typename T, int V, int NC, int L>
int launch_dot(const ThinArgs& p, int64_t sms, cudaStream_t stream) {
  constexpr int kMany = NC <= 2 ? 4 : 2, kWarps = kDotThreads / 32;
  const size_t bytes = static_cast<size_t>(NC) * ((p.len + 3) & ~3) * sizeof(float);
  const bool many = p.rows >= sms * kWarps * (32 / L) * kMany;
  const int64_t want = ceil_div(p.rows, kWarps * (32 / L) * (many ? kMany : 1));
  const int64_t cap = sms * (bytes <= 96 * 1024 ? 2 : 1);
  const auto kernel =
      many ? thin_dot_kernel<T, V, NC, L, kMany> : thin_dot_kernel<T, V, NC, L, 1>;
  const int st = allow_smem(reinterpret_cast<const void*>(kernel), bytes);
  if (st == ICTC_OK)
    kernel<<<static_cast<unsigned>(want < cap ? want : cap), kDotThreads, bytes, stream>>>(p);
  return st;
}

template <typename T, int V, int L>
int launch_dot_columns(const ThinArgs& p, int64_t sms, cudaStream_t stream) {
  switch (thin_columns(p.count)) {
    case 1: return launch_dot<T, V, 1, L>(p, sms, stream);
    case 2: return launch_dot<T, V, 2, L>(p, sms, stream);
    case 4: return launch_dot<T, V, 4, L>(p, sms, stream);
    default: return launch_dot<T, V, kThin, L>(p, sms, stream);
  }
}

// Lanes of a row: enough that consecutive lanes read whole sectors, and no more than leave
// each a few accesses, because every row's sums are joined over them (float32 136,107 x 175 x
// 6: 41 us with 4 lanes of 44 accesses, 89 with 32 of 6), unless rows are few (bf16 1,000 x 512
// x 8: 14 us with 4 lanes, on 8 SMs).
template <typename T, int V>
int launch_dot_lanes(const ThinArgs& p, int64_t sms, cudaStream_t stream) {
  const int accesses = p.len / V;
  if (accesses <= 8) return launch_dot_columns<T, V, 1>(p, sms, stream);
  if (accesses < 16 || (accesses < 1024 && p.rows >= sms * 256))
    return launch_dot_columns<T, V, 4>(p, sms, stream);
  return launch_dot_columns<T, V, 32>(p, sms, stream);
}

template <typename T, bool A_MN, bool B_MN>
int run_thin(Thin form, const T* a, int64_t lda, const T* b, int64_t ldb, int64_t m, int64_t n,
             int64_t k, const Epilogue& e, float* partial, cudaStream_t stream) {
  constexpr int kFull = 16 / sizeof(T);
  const int device = current_device();
  const int64_t sms = sm_count(device);
  // strides of A and B along their own index and along the sum
  const int64_t a_i = A_MN ? 1 : lda, a_k = A_MN ? lda : 1;
  const int64_t b_i = B_MN ? 1 : ldb, b_k = B_MN ? ldb : 1;
  ThinArgs p{};
  p.e = e;
  p.e.vec = vec_epilogue<T>(e, n);
  int st = ICTC_OK;
  if (form == Thin::outer) {
    p.small = a; p.small_i = a_i; p.small_c = a_k;
    p.wide = b; p.wide_c = b_k; p.wide_j = b_i;
    p.rows = m; p.width = n;
    p.count = static_cast<int>(k);
    const StripPlan s = plan_strips(m, n, p.e.vec ? 4 : 1, device);
    p.lanes = s.lanes;
    for_thin(p.count, [&](auto nc) {
      const auto kernel =
          p.e.vec ? thin_outer_kernel<T, 4, nc.value> : thin_outer_kernel<T, 1, nc.value>;
      kernel<<<dim3(s.blocks_x, s.blocks_y), kStripThreads, 0, stream>>>(p);
    });
  } else if (form == Thin::dot || form == Thin::dot_swapped) {
    p.swapped = form == Thin::dot_swapped;
    p.big = p.swapped ? b : a;
    p.big_ld = p.swapped ? ldb : lda;
    p.small = p.swapped ? a : b;
    p.small_i = p.swapped ? a_k : b_k;
    p.small_c = p.swapped ? a_i : b_i;
    p.rows = p.swapped ? n : m;
    p.len = static_cast<int>(k);
    p.count = static_cast<int>(p.swapped ? m : n);
    const bool vec =
        k % kFull == 0 && chunk_aligned(p.big, p.big_ld, sizeof(T));
    st = vec ? launch_dot_lanes<T, kFull>(p, sms, stream) : launch_dot_lanes<T, 1>(p, sms, stream);
    if (st != ICTC_OK) return st;
  } else {
    // the operand whose rows the sum runs over, and the few columns of the other
    p.swapped = form == Thin::gram_swapped;
    p.big = p.swapped ? a : b;
    p.big_ld = p.swapped ? lda : ldb;
    p.small = p.swapped ? b : a;
    p.small_i = p.swapped ? b_k : a_k;
    p.small_c = p.swapped ? b_i : a_i;
    p.rows = k;
    p.width = p.swapped ? m : n;
    p.count = static_cast<int>(p.swapped ? n : m);
    p.partial = partial;
    const bool vec = p.width % kFull == 0 && chunk_aligned(p.big, p.big_ld, sizeof(T));
    const StripPlan s = plan_strips(p.rows, p.width, vec ? kFull : 1, device);
    p.lanes = s.lanes;
    for_thin(p.count, [&](auto nc) {
      const auto kernel =
          vec ? thin_gram_kernel<T, kFull, nc.value> : thin_gram_kernel<T, 1, nc.value>;
      kernel<<<dim3(s.blocks_x, s.blocks_y), kStripThreads, 0, stream>>>(p);
    });
    const cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return cuda_fail(err, "thin linear product launch");
    T* out = static_cast<T*>(e.out);
    column_total_kernel<T><<<dim3(static_cast<unsigned>(ceil_div(m * n, 32))),
                             dim3(32, kColumnLanes), 0, stream>>>(partial, partial, out, out,
                                                                  s.blocks_y, m * n);
  }
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? ICTC_OK : cuda_fail(err, "thin linear product launch");
}

// C = epilogue(A B^T); `partial` holds product_bytes().
template <typename T, bool A_MN, bool B_MN>
int run_product(const T* a, int64_t lda, const T* b, int64_t ldb, int64_t m, int64_t n, int64_t k,
                Epilogue e, float* partial, bool tiles, cudaStream_t stream) {
  const int device = current_device();
  e.vec = vec_epilogue<T>(e, n);
  const auto join = [&](int splits) {
    const int64_t blocks = ceil_div(m * ceil_div(n, 4), 256);
    const int64_t cap = static_cast<int64_t>(sm_count(device)) * 8;
    e.partial = partial;
    join_splits_kernel<T><<<static_cast<unsigned>(blocks < cap ? blocks : cap), 256, 0, stream>>>(
        e, m, n, splits);
    const cudaError_t err = cudaGetLastError();
    return err == cudaSuccess ? ICTC_OK : cuda_fail(err, "linear split join launch");
  };
  if constexpr (B_MN) {  // a gradient (the forward's form is in its plan)
    if (const Thin form = thin_form(A_MN, B_MN, m, n, k, tiles); form != Thin::none)
      return run_thin<T, A_MN, B_MN>(form, a, lda, b, ldb, m, n, k, e, partial, stream);
  }
  if constexpr (sizeof(T) == 2) {
    const PairPlan q = plan_pair(m, n, k, device);
    OperandMaps maps;
    if (q.ok && use_pair(m, n, k) && chunk_aligned(a, lda, 2) && chunk_aligned(b, ldb, 2)) {
      constexpr bool kBf16 = std::is_same_v<T, __nv_bfloat16>;
      const bool mapped =
          encode_matrix_map(a, 2, kBf16, A_MN ? m : k, A_MN ? k : m, lda * 2, 64, A_MN ? 64 : 128,
                            &maps.a) == 0 &&
          encode_matrix_map(b, 2, kBf16, B_MN ? n : k, B_MN ? k : n, ldb * 2, 64,
                            B_MN ? 64 : q.bn / 2, &maps.b) == 0;
      if (mapped) {
        ProductArgs p{};
        p.m = m; p.n = n; p.k = k;
        p.tiles_m = q.tiles_m; p.tiles_n = q.tiles_n;
        p.splits = q.splits; p.chunks = q.chunks; p.chunks_per_split = q.chunks_per_split;
        p.e = e;
        p.e.partial = q.splits > 1 ? partial : nullptr;
        const int st = q.bn == 256 ? launch_pair<T, A_MN, B_MN, 256>(maps, p, device, stream)
                                   : launch_pair<T, A_MN, B_MN, 128>(maps, p, device, stream);
        return st != ICTC_OK || q.splits == 1 ? st : join(q.splits);
      }
    }
  }
  ProductArgs p{};
  p.a = a; p.b = b;
  p.m = m; p.n = n; p.k = k;
  p.lda = lda; p.ldb = ldb;
  p.vec_a = chunk_aligned(a, lda, sizeof(T));
  p.vec_b = chunk_aligned(b, ldb, sizeof(T));
  const auto take = [&](const Split& s) {
    p.tiles_m = s.tiles_m; p.tiles_n = s.tiles_n;
    p.splits = s.splits; p.chunks = s.chunks; p.chunks_per_split = s.chunks_per_split;
    e.partial = s.splits > 1 ? partial : nullptr;
    p.e = e;
  };
  if constexpr (sizeof(T) == 4) {
    const Split s = plan_product(m, n, k, true, device);
    if (!s.fits) return fail(ICTC_ERR_UNSUPPORTED, "linear: a dimension is too large");
    take(s);
    OperandMaps maps;
    if (p.vec_a && p.vec_b && m < (1ll << 31) && n < (1ll << 31) && k < (1ll << 31) &&
        encode_matrix_map(a, 4, false, A_MN ? m : k, A_MN ? k : m, lda * 4, A_MN ? 128 : kCutK,
                          A_MN ? kCutK : 128, &maps.a) == 0 &&
        encode_matrix_map(b, 4, false, B_MN ? n : k, B_MN ? k : n, ldb * 4, B_MN ? s.bn : kCutK,
                          B_MN ? kCutK : s.bn, &maps.b) == 0) {
      const int st = s.bn == 64 ? launch_cut<A_MN, B_MN, 64>(maps, p, device, stream)
                                : launch_cut<A_MN, B_MN, 128>(maps, p, device, stream);
      return st != ICTC_OK || s.splits == 1 ? st : join(s.splits);
    }
  }
  // A float32 tile is 64 columns wide: the cut parts of a wider one do not fit a producer's
  // registers.  (More tiles are never more splits, for which `partial` has room.)
  const Split s = plan_product(m, n, k, sizeof(T) == 4, device, sizeof(T) == 4 ? 64 : 128);
  if (!s.fits) return fail(ICTC_ERR_UNSUPPORTED, "linear: a dimension is too large");
  take(s);
  int st;
  if constexpr (sizeof(T) == 4)
    st = launch_product<T, A_MN, B_MN, 64>(p, device, stream);
  else
    st = s.bn == 64 ? launch_product<T, A_MN, B_MN, 64>(p, device, stream)
                    : launch_product<T, A_MN, B_MN, 128>(p, device, stream);
  return st != ICTC_OK || s.splits == 1 ? st : join(s.splits);
}

template <typename T, int V>
int launch_few_rows(const T* x, int64_t ldx, const T* w, int64_t ldw, int64_t rows, int64_t n,
                    int64_t k, const Epilogue& e, cudaStream_t stream) {
  const int64_t sms = sm_count(current_device());
  // all eight warps of a CTA share a column while that still gives every SM work
  const int share = n <= sms * 16 ? 8 : 1;
  const int64_t want = ceil_div(n, 8 / share);
  const unsigned grid = static_cast<unsigned>(want < sms * 8 ? want : sms * 8);
  if (rows == 1)
    few_rows_kernel<T, 1, V><<<grid, kRowThreads, 0, stream>>>(x, ldx, w, ldw, rows, n, k, share, e);
  else
    few_rows_kernel<T, 4, V><<<grid, kRowThreads, 0, stream>>>(x, ldx, w, ldw, rows, n, k, share, e);
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? ICTC_OK : cuda_fail(err, "linear few-row launch");
}

constexpr int64_t kFewRows = 4;

// ------------------------------------------------------------------- plan of a call

// What a call's pointers and strides allow (ICTC_LINEAR_ALIGNED, ICTC_LINEAR_PACKED).
int32_t layout_of(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* g,
                  int64_t ldg, const void* preact, int64_t m, int64_t n, int64_t k, size_t size) {
  int32_t flags = 0;
  if (chunk_aligned(x, ldx, size) && chunk_aligned(w, ldw, size) &&
      (!g || chunk_aligned(g, ldg, size)))
    flags |= ICTC_LINEAR_ALIGNED;
  if (aligned(x, 16) && (ldx == k || m <= 1) &&
      (!g || (aligned(g, 16) && (ldg == n || m <= 1) && aligned(preact, 16))))
    flags |= ICTC_LINEAR_PACKED;
  return flags;
}

// Byte offsets of the workspace's parts, and its size.
struct LinearPlan {
  bool few, narrow, align;
  bool tiles;  // 16-bit operands that TMA can address
  Thin thin;   // the forward's
  size_t d, x, w, g, columns, partial, total;
};

constexpr int64_t kSlopeParts = 296;

// Most outputs for which the backward of a thin layer leaves the narrow kernel.  That has two
// launches and a fixed time a tile (with SiLU, kernel times of 1,048,576 rows: 223 us float32,
// 150 bf16; 370 and 297 of a million rows that are not whole blocks); the thin forms have five
// and read d for each product: 8 x 8 66 and 59 us, 22 x 1 93 and 84, 61 x 8 294 (narrow 486),
// 8 x 64 348 and 250 (narrow 237 and 148), 7 x 61 450 (narrow 369).
constexpr int64_t kThinOutputs = 24;

LinearPlan plan_linear(int64_t m, int64_t n, int64_t k, int dtype, int activation, int32_t layout,
                       bool backward, int device) {
  LinearPlan b{};
  const size_t size = dtype_size(dtype);
  const int64_t full = static_cast<int64_t>(16 / size);
  const bool rows_aligned = layout & ICTC_LINEAR_ALIGNED;
  b.tiles = size == 2 && rows_aligned;
  // both products of the backward are thin: no operand is copied to aligned rows
  const bool thin = backward && (n <= kThin || m <= kThin || (k <= kThin && dot_fits(m, n, k)));
  b.narrow = (layout & ICTC_LINEAR_PACKED) && n <= kNarrow && k <= kNarrow && m <= (1ll << 36);
  if (!backward) {
    b.few = m <= kFewRows && rows_aligned && k % full == 0;
    if (!b.few) b.thin = thin_form(false, false, m, n, k, b.tiles);
    // a few rows over a weight that few_rows_kernel and TMA would read by elements
    if (!b.few && b.thin == Thin::none && m <= kThin && (m <= kFewRows || !rows_aligned) &&
        dot_fits(n, k, m))
      b.thin = Thin::dot_swapped;
    if (b.thin == Thin::none) b.few = m <= kFewRows;
    b.narrow = b.narrow && !b.few && b.thin == Thin::none;
  } else if (thin && n <= kThinOutputs &&
             m > 2 * kNarrowTile * static_cast<int64_t>(sm_count(device))) {
    b.narrow = false;
  }
  b.align = !rows_aligned && b.thin == Thin::none && !thin && worth_aligning(m, n, k);
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    const size_t here = at;
    at += align_up(bytes, 256);
    return here;
  };
  const auto rows = [&](int64_t r, int64_t width) {
    return static_cast<size_t>(r) * aligned_pitch(width, size) * size;
  };
  if (b.few || b.thin != Thin::none) return b;
  if (b.narrow) {
    if (backward)
      b.partial = take(static_cast<size_t>(sm_count(device)) * (n * k + n) * sizeof(float));
    b.total = at;
    return b;
  }
  const bool slope = backward && activation != ICTC_ACT_NONE;
  if (slope) b.d = take(rows(m, n));
  if (b.align) {
    b.x = take(rows(m, k));
    b.w = take(rows(n, k));
    if (backward && !slope) b.g = take(rows(m, n));
  }
  if (backward) {
    b.columns = take(static_cast<size_t>(m < kSlopeParts ? m : kSlopeParts) * n * sizeof(float));
    const size_t one = product_bytes(false, true, m, k, n, dtype, device);
    const size_t other = product_bytes(true, true, n, k, m, dtype, device);
    b.partial = take(one > other ? one : other);
  } else {
    b.partial = take(split_bytes(m, n, k, dtype, device));
  }
  b.total = at;
  return b;
}

template <typename T>
int run_narrow_forward(const T* x, const T* w, int64_t ldw, Epilogue e, int64_t m, int64_t n,
                       int64_t k, cudaStream_t stream) {
  NarrowArgs p{};
  p.x = x; p.w = w;
  p.m = m; p.ldw = ldw;
  p.n = static_cast<int>(n); p.k = static_cast<int>(k);
  p.tiles = static_cast<int>(ceil_div(m, kNarrowTile));
  e.vec = vec_epilogue<T>(e, n);
  p.e = e;
  const int sms = sm_count(current_device());
  const int grid = p.tiles < sms ? p.tiles : sms;
  int st = ICTC_OK;
  const bool plain = k * sizeof(T) % 16 == 0;
  for_activation(e.activation, [&](auto act) {
    const auto kernel = plain ? narrow_forward_kernel<T, act.value, true>
                              : narrow_forward_kernel<T, act.value, false>;
    st = allow_smem(reinterpret_cast<const void*>(kernel), kNarrowForwardSmem<T>);
    if (st == ICTC_OK) kernel<<<grid, kNarrowThreadsL, kNarrowForwardSmem<T>, stream>>>(p);
  });
  if (st != ICTC_OK) return st;
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? ICTC_OK : cuda_fail(err, "narrow linear forward launch");
}

template <typename T>
int run_narrow_backward(const T* x, const T* w, int64_t ldw, const float* preact, const T* g,
                        T* dx, T* dw, T* db, float* partial, int64_t m, int64_t n, int64_t k,
                        int activation, cudaStream_t stream) {
  NarrowArgs p{};
  p.x = x; p.w = w; p.g = g; p.preact = preact;
  p.m = m; p.ldw = ldw;
  p.n = static_cast<int>(n); p.k = static_cast<int>(k);
  p.tiles = static_cast<int>(ceil_div(m, kNarrowTile));
  p.partial = dw || db ? partial : nullptr;
  p.e.out = dx;
  p.e.vec = vec_epilogue<T>(p.e, k);
  const int sms = sm_count(current_device());
  const int grid = p.tiles < sms ? p.tiles : sms;
  int st = ICTC_OK;
  const bool plain = k * sizeof(T) % 16 == 0 && n * sizeof(T) % 16 == 0;
  for_activation(activation, [&](auto act) {
    const auto kernel = plain ? narrow_backward_kernel<T, act.value, true>
                              : narrow_backward_kernel<T, act.value, false>;
    st = allow_smem(reinterpret_cast<const void*>(kernel), kNarrowBackwardSmem<T>);
    if (st == ICTC_OK) kernel<<<grid, kNarrowThreadsL, kNarrowBackwardSmem<T>, stream>>>(p);
  });
  if (st != ICTC_OK) return st;
  cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return cuda_fail(err, "narrow linear backward launch");
  if (!p.partial) return ICTC_OK;
  const int nk = p.n * p.k;
  narrow_total_kernel<T><<<static_cast<unsigned>(ceil_div(nk + p.n, 32)), dim3(32, kColumnLanes),
                           0, stream>>>(partial, dw, db, grid, nk, p.n);
  err = cudaGetLastError();
  return err == cudaSuccess ? ICTC_OK : cuda_fail(err, "narrow linear column sum launch");
}

template <typename T>
int run_linear_forward(const void* x, int64_t ldx, const void* w, int64_t ldw, Epilogue e,
                       unsigned char* workspace, const LinearPlan& plan, int64_t m, int64_t n,
                       int64_t k, cudaStream_t stream) {
  const T* xt = static_cast<const T*>(x);
  const T* wt = static_cast<const T*>(w);
  if (plan.few) {
    constexpr int kFull = 16 / sizeof(T);
    if (k % kFull == 0 && chunk_aligned(x, ldx, sizeof(T)) && chunk_aligned(w, ldw, sizeof(T)))
      return launch_few_rows<T, kFull>(xt, ldx, wt, ldw, m, n, k, e, stream);
    return launch_few_rows<T, 1>(xt, ldx, wt, ldw, m, n, k, e, stream);
  }
  if (plan.narrow) return run_narrow_forward<T>(xt, wt, ldw, e, m, n, k, stream);
  if (plan.thin != Thin::none)
    return run_thin<T, false, false>(plan.thin, xt, ldx, wt, ldw, m, n, k, e, nullptr, stream);
  if (plan.align) {
    int st = align_operand(&xt, &ldx, m, k, workspace + plan.x, stream);
    if (st == ICTC_OK) st = align_operand(&wt, &ldw, n, k, workspace + plan.w, stream);
    if (st != ICTC_OK) return st;
  }
  return run_product<T, false, false>(xt, ldx, wt, ldw, m, n, k, e,
                                      reinterpret_cast<float*>(workspace + plan.partial),
                                      plan.tiles, stream);
}

struct SlopePlan {
  int vec, lanes;
  unsigned blocks_x, blocks_y;
};

SlopePlan plan_slope(int64_t m, int64_t n, int vec) {
  SlopePlan s{};
  s.vec = vec;
  const int64_t units = ceil_div(n, vec);
  int lanes = 1;
  while (lanes < 32 && lanes < units) lanes *= 2;
  s.lanes = lanes;
  s.blocks_x = static_cast<unsigned>(ceil_div(units, lanes));
  const int64_t row_blocks = ceil_div(m, 256 / lanes);
  int64_t y = ceil_div(static_cast<int64_t>(sm_count(current_device())) * 8, s.blocks_x);
  if (y > kSlopeParts) y = kSlopeParts;
  if (y > row_blocks) y = row_blocks;
  // short sums are finished where they are formed: up to eight rounds of four rows a thread
  // cost less than the launch that joins parts (1,000 x 72 had 32 rounds: 24 us)
  if (row_blocks <= 32) y = 1;
  s.blocks_y = static_cast<unsigned>(y < 1 ? 1 : y);
  return s;
}

template <typename T>
int run_linear_backward(const void* x, int64_t ldx, const void* w, int64_t ldw,
                        const float* preact, const void* g, int64_t ldg, void* dx, void* dw,
                        void* db, unsigned char* workspace, const LinearPlan& plan, int64_t m,
                        int64_t n, int64_t k, int activation, cudaStream_t stream) {
  const T* xt = static_cast<const T*>(x);
  const T* wt = static_cast<const T*>(w);
  const T* d = static_cast<const T*>(g);
  float* partial = reinterpret_cast<float*>(workspace + plan.partial);
  if (plan.narrow)
    return run_narrow_backward<T>(xt, wt, ldw, preact, d, static_cast<T*>(dx),
                                  static_cast<T*>(dw), static_cast<T*>(db), partial, m, n, k,
                                  activation, stream);
  int64_t ldd = ldg;
  const bool slope = activation != ICTC_ACT_NONE;
  T* d_out = slope ? reinterpret_cast<T*>(workspace + plan.d) : nullptr;
  const int64_t d_pitch = aligned_pitch(n, sizeof(T));
  float* columns = db ? reinterpret_cast<float*>(workspace + plan.columns) : nullptr;
  if (slope || db) {
    constexpr int kFull = 16 / sizeof(T);
    const bool vec = n % kFull == 0 && chunk_aligned(g, ldg, sizeof(T)) && aligned(preact, 16);
    const SlopePlan s = plan_slope(m, n, vec ? kFull : 1);
    const dim3 grid(s.blocks_x, s.blocks_y);
    T* db_out = s.blocks_y == 1 ? static_cast<T*>(db) : nullptr;  // no partial rows to join
    for_activation(activation, [&](auto act) {
      if (vec)
        slope_kernel<T, kFull, act.value><<<grid, 256, 0, stream>>>(d, ldg, preact, d_out, d_pitch,
                                                                    columns, db_out, m, n, s.lanes);
      else
        slope_kernel<T, 1, act.value><<<grid, 256, 0, stream>>>(d, ldg, preact, d_out, d_pitch,
                                                                columns, db_out, m, n, s.lanes);
    });
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "linear slope launch");
    if (db && !db_out) {
      column_total_kernel<T><<<dim3(static_cast<unsigned>(ceil_div(n, 32))),
                               dim3(32, kColumnLanes), 0, stream>>>(
          columns, columns, static_cast<T*>(db), static_cast<T*>(db), s.blocks_y, n);
      e = cudaGetLastError();
      if (e != cudaSuccess) return cuda_fail(e, "linear column sum launch");
    }
    if (slope) {
      d = d_out;
      ldd = d_pitch;
    }
  }
  if (plan.align) {
    int st = ICTC_OK;
    if (!slope && (dx || dw)) st = align_operand(&d, &ldd, m, n, workspace + plan.g, stream);
    if (st == ICTC_OK && dx) st = align_operand(&wt, &ldw, n, k, workspace + plan.w, stream);
    if (st == ICTC_OK && dw) st = align_operand(&xt, &ldx, m, k, workspace + plan.x, stream);
    if (st != ICTC_OK) return st;
  }
  Epilogue e{};
  if (dx) {
    e.out = dx;
    const int st =
        run_product<T, false, true>(d, ldd, wt, ldw, m, k, n, e, partial, plan.tiles, stream);
    if (st != ICTC_OK) return st;
  }
  if (dw) {
    e.out = dw;
    return run_product<T, true, true>(d, ldd, xt, ldx, n, k, m, e, partial, plan.tiles, stream);
  }
  return ICTC_OK;
}

int check_linear(int64_t m, int64_t n, int64_t k, int32_t dtype, int32_t activation) {
  if (m < 0 || n < 1 || k < 1)
    return fail(ICTC_ERR_INVALID,
                "linear needs rows >= 0 and in, out >= 1, got %lld rows, in %lld, out %lld",
                static_cast<long long>(m), static_cast<long long>(k), static_cast<long long>(n));
  if (!known_dtype(dtype)) return fail(ICTC_ERR_INVALID, "unknown dtype code %d", dtype);
  if (activation < ICTC_ACT_NONE || activation > ICTC_ACT_GELU_TANH)
    return fail(ICTC_ERR_INVALID, "unknown activation code %d", activation);
  return ICTC_OK;
}

}  // namespace

int dense_take_device_error(int* code) {
  cudaError_t e;
  if (take_unit_device_error(code, &e) != 0) return cuda_fail(e, "linear device error flag");
  return ICTC_OK;
}

}  // namespace ictc

using namespace ictc;

extern "C" int32_t ictc_o2_linear_workspace(int64_t rows, int64_t in, int64_t out, int32_t dtype,
                                            int32_t activation, int32_t layout, int32_t device,
                                            size_t* forward_bytes, size_t* backward_bytes) {
  const int st = check_linear(rows, out, in, dtype, activation);
  if (st != ICTC_OK) return st;
  if (!forward_bytes || !backward_bytes) return fail(ICTC_ERR_INVALID, "null output");
  *forward_bytes = *backward_bytes = 0;
  if (rows == 0) return ICTC_OK;
  *forward_bytes =
      plan_linear(rows, out, in, dtype, activation, layout, false, device).total;
  *backward_bytes =
      plan_linear(rows, out, in, dtype, activation, layout, true, device).total;
  return ICTC_OK;
}

extern "C" int32_t ictc_o2_linear_forward(const void* x, int64_t x_stride, const void* weight,
                                          int64_t weight_stride, const void* bias,
                                          const void* residual, int64_t residual_stride, void* y,
                                          float* preact, void* workspace, size_t workspace_bytes,
                                          int64_t rows, int64_t in, int64_t out, int32_t dtype,
                                          int32_t activation, void* stream) {
  const int st = check_linear(rows, out, in, dtype, activation);
  if (st != ICTC_OK) return st;
  if (rows == 0) return ICTC_OK;
  if (!x || !weight || !y) return fail(ICTC_ERR_INVALID, "null pointer");
  if (x_stride < 0 || weight_stride < 0 || residual_stride < 0)
    return fail(ICTC_ERR_INVALID, "negative row stride");
  const int32_t layout = layout_of(x, x_stride, weight, weight_stride, nullptr, 0, nullptr, rows,
                                   out, in, dtype_size(dtype));
  const LinearPlan plan =
      plan_linear(rows, out, in, dtype, activation, layout, false, current_device());
  if (plan.total > 0 &&
      (!workspace || workspace_bytes < plan.total || !aligned(workspace, 256)))
    return fail(ICTC_ERR_WORKSPACE, "workspace has %zu bytes, needs %zu (256-byte aligned)",
                workspace ? workspace_bytes : 0, plan.total);
  Epilogue e{};
  e.bias = bias;
  e.residual = residual;
  e.residual_stride = residual_stride;
  e.preact = preact;
  e.out = y;
  e.activation = activation;
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define ICTC_LINEAR_FORWARD(T) \
  return run_linear_forward<T>(x, x_stride, weight, weight_stride, e, ws, plan, rows, out, in, s)
  if (dtype == ICTC_DTYPE_F32) ICTC_LINEAR_FORWARD(float);
  if (dtype == ICTC_DTYPE_BF16) ICTC_LINEAR_FORWARD(__nv_bfloat16);
  ICTC_LINEAR_FORWARD(__half);
#undef ICTC_LINEAR_FORWARD
}

extern "C" int32_t ictc_o2_linear_backward(
    const void* x, int64_t x_stride, const void* weight, int64_t weight_stride,
    const float* preact, const void* grad_output, int64_t grad_stride, void* grad_x,
    void* grad_weight, void* grad_bias, void* workspace, size_t workspace_bytes, int64_t rows,
    int64_t in, int64_t out, int32_t dtype, int32_t activation, void* stream) {
  const int st = check_linear(rows, out, in, dtype, activation);
  if (st != ICTC_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    cudaError_t e = cudaSuccess;
    if (grad_weight)
      e = cudaMemsetAsync(grad_weight, 0, static_cast<size_t>(out) * in * dtype_size(dtype), s);
    if (e == cudaSuccess && grad_bias)
      e = cudaMemsetAsync(grad_bias, 0, static_cast<size_t>(out) * dtype_size(dtype), s);
    return e == cudaSuccess ? ICTC_OK : cuda_fail(e, "linear gradient clear");
  }
  if (!grad_x && !grad_weight && !grad_bias) return ICTC_OK;
  if (!x || !weight || !grad_output || (activation != ICTC_ACT_NONE && !preact))
    return fail(ICTC_ERR_INVALID, "null pointer");
  if (x_stride < 0 || weight_stride < 0 || grad_stride < 0)
    return fail(ICTC_ERR_INVALID, "negative row stride");
  const int32_t layout =
      layout_of(x, x_stride, weight, weight_stride, grad_output, grad_stride,
                activation == ICTC_ACT_NONE ? nullptr : preact, rows, out, in, dtype_size(dtype));
  const LinearPlan plan =
      plan_linear(rows, out, in, dtype, activation, layout, true, current_device());
  if (plan.total > 0 &&
      (!workspace || workspace_bytes < plan.total || !aligned(workspace, 256)))
    return fail(ICTC_ERR_WORKSPACE, "workspace has %zu bytes, needs %zu (256-byte aligned)",
                workspace ? workspace_bytes : 0, plan.total);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
#define ICTC_LINEAR_BACKWARD(T)                                                               \
  return run_linear_backward<T>(x, x_stride, weight, weight_stride, preact, grad_output,       \
                                grad_stride, grad_x, grad_weight, grad_bias, ws, plan, rows, out, \
                                in, activation, s)
  if (dtype == ICTC_DTYPE_F32) ICTC_LINEAR_BACKWARD(float);
  if (dtype == ICTC_DTYPE_BF16) ICTC_LINEAR_BACKWARD(__nv_bfloat16);
  ICTC_LINEAR_BACKWARD(__half);
#undef ICTC_LINEAR_BACKWARD
}
