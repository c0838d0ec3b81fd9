// Fifth-generation tensor core (tcgen05) helpers for sm_100a: TMEM allocation, matrix
// and instruction descriptors, MMA issue and TMEM loads, one CTA per MMA.
//
// Operand tiles live in shared memory as rows of 128 bytes (64 16-bit elements) whose
// 16-byte chunks are XOR-swizzled by the row's index modulo 8 (the 128-byte swizzle):
// chunk c of row r sits at r * 128 + ((c ^ (r & 7)) << 4).  The same bytes serve both
// operand orders:
//   K-major   a row is one M (or N) index, its 64 elements run along K;
//   MN-major  a row is one K index, its 64 elements run along M (or N); tiles wider than
//             64 are blocks of [K rows][128 bytes] one after the other.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "tma.cuh"

namespace ictc {

// Byte offset of 16-byte chunk `c` of 128-byte row `r`.
__device__ __forceinline__ uint32_t swizzled(uint32_t r, uint32_t c) {
  return r * 128 + ((c ^ (r & 7)) << 4);
}

// The bf16 parts of two float32 values, eight significant bits each by truncation (the
// three add up to a finite value exactly), the first value in the low half.
__device__ __forceinline__ void cut_pair(float x0, float x1, uint32_t (&part)[3]) {
  const uint32_t u0 = __float_as_uint(x0), u1 = __float_as_uint(x1);
  part[0] = __byte_perm(u0, u1, 0x7632);
  // x - (leading part): the sign is flipped on the integer side, the pair added at once
  const float2 r = __fadd2_rn(make_float2(x0, x1),
                              make_float2(__uint_as_float((u0 & 0xffff0000u) ^ 0x80000000u),
                                          __uint_as_float((u1 & 0xffff0000u) ^ 0x80000000u)));
  const uint32_t v0 = __float_as_uint(r.x), v1 = __float_as_uint(r.y);
  part[1] = __byte_perm(v0, v1, 0x7632);
  const float2 s = __fadd2_rn(r, make_float2(__uint_as_float((v0 & 0xffff0000u) ^ 0x80000000u),
                                             __uint_as_float((v1 & 0xffff0000u) ^ 0x80000000u)));
  part[2] = __byte_perm(__float_as_uint(s.x), __float_as_uint(s.y), 0x7632);
}

// An element of a float32 product from its sums of leading parts (a1 b1) and of the others.
// An infinity is its own leading part (a NaN too), its other parts are NaN: the first sum
// alone has what a product in order gives, with its sign, and the NaN of the others is
// replaced by a finite value.
__device__ __forceinline__ float join_parts(float leading, float others) {
  return leading + fmaxf(others, -3.402823466e38f);
}

// Shared-memory matrix descriptor, 128-byte swizzle.  Groups of eight 128-byte rows are
// `stride` bytes apart; `leading` is the distance of the 64-element blocks of an
// MN-major operand (unused for K-major ones).
__device__ __forceinline__ uint64_t matrix_descriptor(uint32_t addr, uint32_t leading,
                                                      uint32_t stride) {
  return static_cast<uint64_t>((addr & 0x3ffff) >> 4) |
         (static_cast<uint64_t>(leading >> 4) << 16) |
         (static_cast<uint64_t>(stride >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// Instruction descriptor of kind::f16: float32 accumulators, A and B both bf16 or both
// f16, each K-major (0) or MN-major (1).
__host__ __device__ constexpr uint32_t mma_descriptor(bool bf16, bool a_mn, bool b_mn, int m,
                                                      int n) {
  return (1u << 4) | (static_cast<uint32_t>(bf16) << 7) | (static_cast<uint32_t>(bf16) << 10) |
         (static_cast<uint32_t>(a_mn) << 15) | (static_cast<uint32_t>(b_mn) << 16) |
         (static_cast<uint32_t>(n / 8) << 17) | (static_cast<uint32_t>(m / 16) << 24);
}

// Whole warp: `columns` TMEM columns (a power of two >= 32); the address lands in *out.
__device__ __forceinline__ void tmem_alloc(uint32_t* out, uint32_t columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                   smem_addr(out)),
               "r"(columns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns)
               : "memory");
}

// One thread: D[tmem] (+)= A B over one K step of 16; `add` false overwrites D.
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t desc,
                                        bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(desc), "r"(static_cast<uint32_t>(add))
      : "memory");
}

// The same thread: one arrival on `bar` when every MMA issued so far has finished.
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
          smem_addr(bar))
      : "memory");
}

__device__ __forceinline__ void tcgen05_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}

__device__ __forceinline__ void tcgen05_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// Orders this thread's shared-memory stores before later reads by the MMA (async proxy).
__device__ __forceinline__ void fence_proxy_async() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Whole warp: 16 consecutive columns of the warp's 32 TMEM lanes; lane l gets lane l's.
// The values are valid after tmem_load_wait().
__device__ __forceinline__ void tmem_load16(uint32_t addr, float (&v)[16]) {
  uint32_t u[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]),
        "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]),
        "=r"(u[14]), "=r"(u[15])
      : "r"(addr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(u[i]);
}

__device__ __forceinline__ void tmem_load_wait() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

}  // namespace ictc
