// The global norm of many tensors, and clipping by it.
//
//   norm = sqrt(sum over all tensors of g^2), or max |g|
//   c = min(1, max_norm / (norm + 1e-6)),  out = c g
//
// Bound by HBM: every value is read for the norm, and where c < 1 (or the result goes
// elsewhere) read again and written.  A launch takes up to 1,024 tensors of mixed types,
// their addresses and sizes among its arguments, so nothing is copied to the device and a
// captured call holds all it needs.  Work is cut into chunks of 32 KB that are dealt out to
// groups of 256 threads in order, and sums are added up in that order, so that results do not
// depend on scheduling.
//
// Two launches: every CTA leaves its sum in the workspace; every CTA of the second adds those
// up and scales its chunks, from the last to the first, which are still in L2.  Up to
// kClusterChunks chunks are one launch of a cluster, whose CTAs read each other's sums from
// shared memory.  268,435,456 float32 values: norm 170 us (6.3 TB/s), scaling 340 us (6.3); bf16
// norm 83 us (6.5).  300 tensors of 40 million values: 31 and 34 us.  16 tensors of 24,768: 5.8
// us in all.
//
// Squares are added in float32 over the 16 bytes of a load and in float64 beyond.  Where
// such a short sum leaves float32's safe range it is taken again in float64, so the norm is
// finite wherever float32 holds it, and small gradients do not vanish.
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "common.cuh"
#include "dense_pair.cuh"
#include "dense_types.cuh"

namespace ictc {
namespace {

constexpr int kThreads = 256;  // of a group that takes a chunk
constexpr int kUnits = 8;      // 16-byte units of a chunk per thread
constexpr int kChunkBytes = kThreads * kUnits * 16;
constexpr int kBlocksPerSm = 2;  // as many as run at a time, by their registers
constexpr int kClusterCtas = 8, kClusterGroups = 2;  // groups of a CTA
constexpr int kClusterChunks = 128;
constexpr int kMostTensors = 1024;  // of a launch: 29 bytes each of its 32,764 of arguments

enum Kind { kTwoNorm = ICTC_GRAD_NORM_2, kMaxNorm = ICTC_GRAD_NORM_MAX };

// Chunk c of a tensor is the c-th whole chunk counted from the 16-byte boundary at or below
// its first element (its first `shift` elements are not the tensor's).
template <int N>
struct Tensors {
  const void* in[N];
  void* out[N];
  int64_t count[N];
  int first[N + 1];  // chunks before each tensor
  uint8_t dtype[N];
  int tensors;
  bool in_place;  // every out is its in
};

// A chunk of a launch: chunk number `chunk` of a tensor.
struct Item {
  const void* in;
  void* out;
  int64_t count, chunk;
  int dtype;
};

template <int N>
__device__ __forceinline__ Item item_at(const Tensors<N>& list, int chunk) {
  int low = 0, high = list.tensors;  // first[low] <= chunk < first[high]
  while (high - low > 1) {
    const int mid = (low + high) >> 1;
    if (list.first[mid] <= chunk) low = mid;
    else high = mid;
  }
  return {list.in[low], list.out[low], list.count[low], chunk - list.first[low], list.dtype[low]};
}

// What a chunk's elements are: the tensor's are [begin, end) of the chunk's.
template <typename T>
struct Chunk {
  const T* in;  // of the chunk's first element, which may not be the tensor's
  int64_t offset;
  int begin, end;
};

template <typename T>
__device__ __forceinline__ Chunk<T> chunk_of(const Item& at) {
  constexpr int kElements = kChunkBytes / sizeof(T);
  const T* base = static_cast<const T*>(at.in);
  const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(base) % 16 / sizeof(T));
  Chunk<T> c;
  c.offset = at.chunk * kElements - shift;
  c.in = base + c.offset;
  c.begin = at.chunk == 0 ? shift : 0;
  const int64_t left = at.count - c.offset;
  c.end = left < kElements ? static_cast<int>(left) : kElements;
  return c;
}

// Calls f(item) for the chunks of the CTA, from the first to the last, or back.  They are found
// ahead, kItems at a time, by a thread each: a search through the arguments costs a miss of the
// constant cache a step, which the chunks would wait for one after the other (300 mixed tensors,
// norm and scaling: 81 us, found ahead 65).
constexpr int kItems = 64;

template <int N, typename F>
__device__ __forceinline__ void for_chunks(const Tensors<N>& list, bool back, const F& f) {
  __shared__ Item items[kItems];
  const int chunks = list.first[list.tensors], step = static_cast<int>(gridDim.x);
  const int first = static_cast<int>(blockIdx.x);
  const int rounds = first < chunks ? (chunks - 1 - first) / step + 1 : 0;
  const int batches = (rounds + kItems - 1) / kItems;
  for (int i = 0; i < batches; ++i) {
    const int base = (back ? batches - 1 - i : i) * kItems;
    const int here = rounds - base < kItems ? rounds - base : kItems;
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < here)
      items[threadIdx.x] = item_at(list, first + (base + static_cast<int>(threadIdx.x)) * step);
    __syncthreads();
    for (int j = 0; j < here; ++j) f(items[back ? here - 1 - j : j]);
  }
}

// The same for a group of a cluster's CTA, which has a few chunks at most: each found as it comes.
template <int N, typename F>
__device__ __forceinline__ void for_chunks_of_group(const Tensors<N>& list, const F& f) {
  const int chunks = list.first[list.tensors];
  for (int c = static_cast<int>(blockIdx.x) * kClusterGroups + threadIdx.x / kThreads; c < chunks;
       c += kClusterCtas * kClusterGroups)
    f(item_at(list, c));
}

template <typename T>
constexpr int kPerUnit = 16 / sizeof(T);

template <typename T>
struct Held {
  Pack<T, kPerUnit<T>> unit[kUnits];
};

// A thread's units of a chunk, every kThreads-th; zeros outside the tensor.  All but a tensor's
// first and last chunk take the first branch, whose loads go out together.
template <typename T>
__device__ __forceinline__ void load_units(const Chunk<T>& c, int thread, Held<T>& h) {
  constexpr int V = kPerUnit<T>;
  using Unit = Pack<T, V>;
  if (c.begin == 0 && c.end == kThreads * kUnits * V) {
#pragma unroll
    for (int i = 0; i < kUnits; ++i)
      h.unit[i] = *reinterpret_cast<const Unit*>(c.in + (i * kThreads + thread) * V);
    return;
  }
  // whole units first, their loads together, then the one at either end
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int at = (i * kThreads + thread) * V;
    h.unit[i] = Unit{};
    if (at >= c.begin && at + V <= c.end) h.unit[i] = *reinterpret_cast<const Unit*>(c.in + at);
  }
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int at = (i * kThreads + thread) * V;
    const bool cut = (at < c.begin && at + V > c.begin) || (at < c.end && at + V > c.end);
    if (cut)
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (at + j >= c.begin && at + j < c.end) h.unit[i].v[j] = c.in[at + j];
  }
}

// A thread's running value: a sum of squares, or the largest |g| as the bits of a
// non-negative float32 (whose order is that of integers, with NaN above infinity).
template <int KIND>
struct Running;

template <>
struct Running<kTwoNorm> {
  double value = 0.0;
  template <typename T>
  __device__ __forceinline__ void add(const Held<T>& h) {
    constexpr int V = kPerUnit<T>;
    float s[kUnits], low = 1.f, total = 0.f;
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      s[i] = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float f = to_float(h.unit[i].v[j]);
        s[i] = fmaf(f, f, s[i]);
      }
      low = fminf(low, s[i]);
      total += s[i];
    }
    // float16's squares stay within 2^-48 and 2^32.  One branch for all units, and all of them
    // unrolled: when the pass still found its chunks one by one, a branch for each, or an index
    // into them, held it at 3.7 TB/s in bf16 where this ran at 5.5 (6.5 since).  A unit of zeros
    // takes the branch: with 9 rows in 10 zero the bf16 norm takes 112 us for 89.
    if constexpr (!std::is_same_v<T, __half>) {
      if (!(low >= 1e-30f && total <= 1e38f)) {  // zeros, too small, too large, infinite, NaN
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
          double d = 0.0;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const double f = to_float(h.unit[i].v[j]);
            d = fma(f, f, d);
          }
          value += d;
        }
        return;
      }
    }
#pragma unroll
    for (int i = 0; i < kUnits; i += 2)
      value += static_cast<double>(s[i]) + static_cast<double>(s[i + 1]);
  }
  __device__ __forceinline__ void join(double other) { value += other; }
  __device__ __forceinline__ double get() const { return value; }
  __device__ __forceinline__ double norm() const { return sqrt(value); }
};

template <>
struct Running<kMaxNorm> {
  uint32_t bits = 0;
  template <typename T>
  __device__ __forceinline__ void add(const Held<T>& h) {
#pragma unroll
    for (int i = 0; i < kUnits; ++i)
#pragma unroll
      for (int j = 0; j < kPerUnit<T>; ++j) {
        const uint32_t b = __float_as_uint(to_float(h.unit[i].v[j])) & 0x7fffffffu;
        bits = b > bits ? b : bits;
      }
  }
  __device__ __forceinline__ void join(double other) {
    const uint32_t b = __float_as_uint(static_cast<float>(other)) & 0x7fffffffu;
    bits = b > bits ? b : bits;
  }
  __device__ __forceinline__ double get() const { return __uint_as_float(bits); }
  __device__ __forceinline__ double norm() const { return __uint_as_float(bits); }
};

// The running value over all threads of the CTA, in a fixed order; every thread gets it.
template <int KIND, int GROUPS = 1>
__device__ __forceinline__ Running<KIND> over_block(Running<KIND> r) {
  constexpr int kWarps = GROUPS * kThreads / 32;
  __shared__ double parts[kWarps];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) r.join(__shfl_xor_sync(0xffffffffu, r.get(), o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = r.get();
  __syncthreads();
  Running<KIND> all;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) all.join(parts[w]);
  return all;
}

template <int KIND, typename T>
__device__ __forceinline__ void add_chunk(const Item& at, int thread, Running<KIND>& r) {
  Held<T> h;
  load_units(chunk_of<T>(at), thread, h);
  r.add(h);
}

template <int KIND>
__device__ __forceinline__ void add_item(const Item& at, int thread, Running<KIND>& r) {
  switch (at.dtype) {
    case ICTC_DTYPE_F32: return add_chunk<KIND, float>(at, thread, r);
    case ICTC_DTYPE_BF16: return add_chunk<KIND, __nv_bfloat16>(at, thread, r);
    default: add_chunk<KIND, __half>(at, thread, r);
  }
}

template <int KIND, int N>
__global__ void __launch_bounds__(kThreads, 2)
    partial_kernel(const __grid_constant__ Tensors<N> list, double* __restrict__ partial) {
  Running<KIND> r;
  for_chunks(list, false, [&](const Item& at) { add_item(at, threadIdx.x, r); });
  r = over_block(r);
  if (threadIdx.x == 0) partial[blockIdx.x] = r.get();
}

template <int KIND>
__device__ __forceinline__ double norm_of(const double* __restrict__ partial, int parts) {
  Running<KIND> r;
  for (int i = threadIdx.x; i < parts; i += kThreads) r.join(partial[i]);
  return over_block(r).norm();
}

template <int KIND>
__global__ void __launch_bounds__(kThreads, 2)
    norm_kernel(const double* __restrict__ partial, int parts, float* __restrict__ norm) {
  const double n = norm_of<KIND>(partial, parts);
  if (threadIdx.x == 0) *norm = static_cast<float>(n);
}

// min(1, max_norm / (norm + 1e-6)), rounded once; NaN stays NaN.
__device__ __forceinline__ float factor_of(double norm, double max_norm) {
  const double q = max_norm / (norm + 1e-6);
  return static_cast<float>(q > 1.0 ? 1.0 : q);
}

template <typename T>
__device__ __forceinline__ void scale_chunk(const Item& at, int thread, float factor) {
  constexpr int V = kPerUnit<T>, kElements = kChunkBytes / sizeof(T);
  const Chunk<T> c = chunk_of<T>(at);
  T* out = static_cast<T*>(at.out) + c.offset;
  if (reinterpret_cast<uintptr_t>(out) % 16 == 0) {
    Held<T> h;
    load_units(c, thread, h);
#pragma unroll
    for (int i = 0; i < kUnits; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j)
        h.unit[i].v[j] = from_float<T>(to_float(h.unit[i].v[j]) * factor);
    if (c.begin == 0 && c.end == kElements) {
#pragma unroll
      for (int i = 0; i < kUnits; ++i)
        *reinterpret_cast<Pack<T, V>*>(out + (i * kThreads + thread) * V) = h.unit[i];
      return;
    }
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int e = (i * kThreads + thread) * V;
      if (e >= c.begin && e + V <= c.end) {
        *reinterpret_cast<Pack<T, V>*>(out + e) = h.unit[i];
      } else if (e + V > c.begin && e < c.end) {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (e + j >= c.begin && e + j < c.end) out[e + j] = h.unit[i].v[j];
      }
    }
  } else {  // boundaries apart: element by element
    constexpr int kAhead = 8;
    for (int e0 = thread; e0 < kElements; e0 += kAhead * kThreads) {
      T v[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int e = e0 + i * kThreads;
        if (e >= c.begin && e < c.end) v[i] = c.in[e];
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int e = e0 + i * kThreads;
        if (e >= c.begin && e < c.end) out[e] = from_float<T>(to_float(v[i]) * factor);
      }
    }
  }
}

__device__ __forceinline__ void scale_item(const Item& at, int thread, float factor) {
  switch (at.dtype) {
    case ICTC_DTYPE_F32: return scale_chunk<float>(at, thread, factor);
    case ICTC_DTYPE_BF16: return scale_chunk<__nv_bfloat16>(at, thread, factor);
    default: scale_chunk<__half>(at, thread, factor);
  }
}

template <int KIND, int N>
__global__ void __launch_bounds__(kThreads, 2)
    scale_kernel(const __grid_constant__ Tensors<N> list, const double* __restrict__ partial,
                 int parts, double max_norm, float* __restrict__ norm) {
  const double n = norm_of<KIND>(partial, parts);
  if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(n);
  const float factor = factor_of(n, max_norm);
  if (factor == 1.f && list.in_place) return;  // they are as they should be
  for_chunks(list, true, [&](const Item& at) { scale_item(at, threadIdx.x, factor); });
}

// All of it in one cluster.
template <int KIND, int N>
__global__ void __cluster_dims__(kClusterCtas, 1, 1)
    __launch_bounds__(kThreads* kClusterGroups)
        cluster_kernel(const __grid_constant__ Tensors<N> list, bool scale, double max_norm,
                       float* __restrict__ norm) {
  __shared__ double sum;
  const int thread = threadIdx.x % kThreads;
  Running<KIND> own;
  for_chunks_of_group(list, [&](const Item& at) { add_item(at, thread, own); });
  own = over_block<KIND, kClusterGroups>(own);
  if (threadIdx.x == 0) sum = own.get();
  cluster_sync();
  Running<KIND> all;
#pragma unroll
  for (int c = 0; c < kClusterCtas; ++c) {
    double part;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(part) : "r"(peer_addr(&sum, c)) : "memory");
    all.join(part);
  }
  const double n = all.norm();
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(n);
  const float factor = factor_of(n, max_norm);
  if (scale && !(factor == 1.f && list.in_place))
    for_chunks_of_group(list, [&](const Item& at) { scale_item(at, thread, factor); });
  cluster_sync();  // no CTA leaves while another may read its sum
}

// ----------------------------------------------------------------------- host side

struct Request {
  const void* const* in;
  void* const* out;  // null: the norm alone
  const int64_t* counts;
  const int32_t* dtypes;
  int64_t tensors;
  double max_norm;
  float* norm;
  double* partial;
  cudaStream_t stream;
};

// The tensors from `at` on that one launch takes, without empty ones.
template <int N>
int64_t fill(const Request& q, int64_t at, Tensors<N>& list) {
  list.tensors = 0;
  list.first[0] = 0;
  list.in_place = q.out != nullptr;
  for (; at < q.tensors && list.tensors < N; ++at) {
    if (q.counts[at] == 0) continue;
    const int64_t size = static_cast<int64_t>(dtype_size(q.dtypes[at]));
    const int64_t shift = static_cast<int64_t>(reinterpret_cast<uintptr_t>(q.in[at]) % 16);
    const int64_t chunks = ceil_div(q.counts[at] * size + shift, kChunkBytes);
    if (list.first[list.tensors] + chunks >= (1ll << 31)) break;
    const int i = list.tensors++;
    list.in[i] = q.in[at];
    list.out[i] = q.out ? q.out[at] : nullptr;
    list.in_place = list.in_place && q.out[at] == q.in[at];
    list.count[i] = q.counts[at];
    list.dtype[i] = static_cast<uint8_t>(q.dtypes[at]);
    list.first[i + 1] = list.first[i] + static_cast<int>(chunks);
  }
  return at;
}

int device_sms() {
  int device = 0;
  return sm_count(cudaGetDevice(&device) == cudaSuccess ? device : 0);
}

template <int N>
unsigned grid_of(const Tensors<N>& list) {
  const int most = device_sms() * kBlocksPerSm, chunks = list.first[list.tensors];
  return static_cast<unsigned>(chunks < 1 ? 1 : chunks < most ? chunks : most);
}

int launched() {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? ICTC_OK : cuda_fail(e, "gradient norm launch");
}

template <int KIND, int N>
int run(const Request& q) {
  static thread_local Tensors<N> list;
  int64_t at = fill(q, 0, list);
  const bool whole = at == q.tensors;  // one launch holds all tensors
  if (whole && list.first[list.tensors] <= kClusterChunks) {
    cluster_kernel<KIND, N><<<kClusterCtas, kThreads * kClusterGroups, 0, q.stream>>>(
        list, q.out != nullptr, q.max_norm, q.norm);
    return launched();
  }
  int parts = 0;
  for (;;) {
    const unsigned grid = grid_of(list);
    partial_kernel<KIND, N><<<grid, kThreads, 0, q.stream>>>(list, q.partial + parts);
    parts += static_cast<int>(grid);
    if (at == q.tensors) break;
    at = fill(q, at, list);
  }
  if (!q.out) {
    norm_kernel<KIND><<<1, kThreads, 0, q.stream>>>(q.partial, parts, q.norm);
    return launched();
  }
  float* norm = q.norm;
  at = whole ? q.tensors : fill(q, 0, list);
  for (;;) {
    scale_kernel<KIND, N><<<grid_of(list), kThreads, 0, q.stream>>>(list, q.partial, parts,
                                                                   q.max_norm, norm);
    if (at == q.tensors) return launched();
    norm = nullptr;
    at = fill(q, at, list);
  }
}

template <int KIND>
int run_sized(const Request& q) {
  return q.tensors <= 16 ? run<KIND, 16>(q) : q.tensors <= 128 ? run<KIND, 128>(q)
                                                              : run<KIND, kMostTensors>(q);
}

// A tensor has at most 2^36 elements, so that a launch takes at least 255 of them before its
// count of chunks leaves its integers.
constexpr int64_t kMostElements = 1ll << 36;

int64_t most_launches(int64_t tensors) { return tensors / 255 + 1; }

size_t workspace_bytes_of(int64_t tensors, int device) {
  return static_cast<size_t>(most_launches(tensors)) * sm_count(device) * kBlocksPerSm *
         sizeof(double);
}

int run_request(const Request& q, int32_t kind, const void* workspace, size_t bytes) {
  if (q.tensors < 0) return fail(ICTC_ERR_INVALID, "negative number of tensors");
  if (kind != kTwoNorm && kind != kMaxNorm) return fail(ICTC_ERR_INVALID, "unknown norm %d", kind);
  if (!q.norm || (q.tensors > 0 && (!q.in || !q.counts || !q.dtypes)))
    return fail(ICTC_ERR_INVALID, "null pointer");
  for (int64_t i = 0; i < q.tensors; ++i) {
    if (q.counts[i] < 0 || q.counts[i] > kMostElements)
      return fail(ICTC_ERR_INVALID, "tensor %lld has %lld elements", static_cast<long long>(i),
                  static_cast<long long>(q.counts[i]));
    if (!known_dtype(q.dtypes[i]))
      return fail(ICTC_ERR_INVALID, "unknown dtype code %d", q.dtypes[i]);
    const uintptr_t size = dtype_size(q.dtypes[i]);
    if (q.counts[i] > 0 &&
        (!q.in[i] || !aligned(q.in[i], size) || (q.out && (!q.out[i] || !aligned(q.out[i], size)))))
      return fail(ICTC_ERR_INVALID, "tensor %lld has a null or misaligned pointer",
                  static_cast<long long>(i));
  }
  int device = 0;
  const cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  const size_t needed = workspace_bytes_of(q.tensors, device);
  if (!workspace || bytes < needed || !aligned(workspace, 16))
    return fail(ICTC_ERR_WORKSPACE, "workspace has %zu bytes, needs %zu (16-byte aligned)",
                workspace ? bytes : 0, needed);
  return kind == kTwoNorm ? run_sized<kTwoNorm>(q) : run_sized<kMaxNorm>(q);
}

}  // namespace
}  // namespace ictc

using namespace ictc;

extern "C" int32_t ictc_o2_grad_norm_workspace(int64_t tensors, int32_t device, size_t* bytes) {
  if (tensors < 0) return fail(ICTC_ERR_INVALID, "negative number of tensors");
  if (!bytes) return fail(ICTC_ERR_INVALID, "null output");
  *bytes = workspace_bytes_of(tensors, device);
  return ICTC_OK;
}

extern "C" int32_t ictc_o2_grad_norm(const void* const* grads, const int64_t* counts,
                                     const int32_t* dtypes, int64_t tensors, int32_t kind,
                                     float* norm, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  const Request q{grads, nullptr, counts, dtypes, tensors, 0.0, norm,
                  static_cast<double*>(workspace), static_cast<cudaStream_t>(stream)};
  return run_request(q, kind, workspace, workspace_bytes);
}

extern "C" int32_t ictc_o2_clip_grads(const void* const* grads, void* const* out,
                                      const int64_t* counts, const int32_t* dtypes,
                                      int64_t tensors, int32_t kind, double max_norm, float* norm,
                                      void* workspace, size_t workspace_bytes, void* stream) {
  if (!(max_norm >= 0.0)) return fail(ICTC_ERR_INVALID, "max_norm must be >= 0");
  if (tensors > 0 && !out) return fail(ICTC_ERR_INVALID, "null pointer");
  static void* const kNone[1] = {nullptr};
  const Request q{grads, out ? out : kNone, counts, dtypes, tensors, max_norm, norm,
                  static_cast<double*>(workspace), static_cast<cudaStream_t>(stream)};
  return run_request(q, kind, workspace, workspace_bytes);
}
