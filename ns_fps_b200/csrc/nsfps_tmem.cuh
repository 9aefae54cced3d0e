// nsfps_tmem.cuh -- the fifth-generation tensor core as the feature operators
// use it: tcgen05.mma issued by one warp of a CTA on shared tiles, results in
// tensor memory.
//
// The issuing calls (mma_*) are made by a whole warp in step, and one elected
// lane issues.  Their operands live in registers that a warp shares; computed
// by one lane alone, every descriptor was moved there first, and a product took
// some 100 cycles to issue.  warp_value() tells the compiler that a value is
// the same in all lanes.
//
// Shared tiles hold rows of 64 16-bit elements (128 bytes) in the 128-byte
// swizzle: 16-byte chunk c of row r lies at r * 128 + ((c ^ (r & 7)) << 4), so
// eight rows are one 1,024-byte pattern.  The same tile is an operand whose
// contraction runs along the rows' elements (K-major) or down the rows
// (MN-major).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace nsfps {

__device__ __forceinline__ uint32_t warp_value(uint32_t x) {
  return __shfl_sync(0xffffffffu, x, 0);
}

__device__ __forceinline__ uint32_t swizzled(uint32_t r, uint32_t c) {
  return r * 128u + ((c ^ (r & 7u)) << 4);
}

// Descriptor of a tile at shared address `at` in the 128-byte swizzle: groups
// of eight rows 1,024 bytes apart; further 64-element columns of an MN-major
// operand `lead` bytes apart.
__device__ __forceinline__ uint64_t tile_desc(uint32_t at, uint32_t lead) {
  return (uint64_t)((at & 0x3ffffu) >> 4) | (uint64_t)((lead >> 4) & 0x3fffu) << 16 |
         (uint64_t)(1024u >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// The tile `bytes` behind (its address stays below the field's 256 KB).
__device__ __forceinline__ uint64_t further(uint64_t desc, uint32_t bytes) {
  return desc + (bytes >> 4);
}

// Instruction descriptor: fp32 accumulator, both operands of type T, M x N.
template <class T>
__device__ constexpr uint32_t mma_desc(uint32_t m, uint32_t n, bool a_mn, bool b_mn);
template <>
__device__ constexpr uint32_t mma_desc<__half>(uint32_t m, uint32_t n, bool a_mn, bool b_mn) {
  return 1u << 4 | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | (n >> 3) << 17 | (m >> 4) << 24;
}
template <>
__device__ constexpr uint32_t mma_desc<__nv_bfloat16>(uint32_t m, uint32_t n, bool a_mn,
                                                      bool b_mn) {
  return mma_desc<__half>(m, n, a_mn, b_mn) | 1u << 7 | 1u << 10;
}

// d (+)= a * b; a and b in shared memory.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t desc,
                                       bool add) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n elect.sync _|q, 0xffffffff;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
      ::"r"(d), "l"(a), "l"(b), "r"(desc), "r"((uint32_t)add)
      : "memory");
}
// The same with a in tensor memory (16-bit elements, two per column).
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t desc,
                                       bool add) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n elect.sync _|q, 0xffffffff;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
      ::"r"(d), "r"(a), "l"(b), "r"(desc), "r"((uint32_t)add)
      : "memory");
}
// The barrier completes when the products issued so far have.
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile(
      "{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(bar)
      : "memory");
}

// (one warp) COLS columns of tensor memory; the address is put at shared `at`.
template <uint32_t COLS>
__device__ __forceinline__ void tmem_alloc(uint32_t at) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(at), "n"(COLS)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
template <uint32_t COLS>
__device__ __forceinline__ void tmem_free(uint32_t addr) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "n"(COLS)
               : "memory");
}
__device__ __forceinline__ void tmem_before_sync() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tmem_after_sync() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// Shared memory written by this thread's copies and stores, for the tensor core.
__device__ __forceinline__ void smem_to_mma() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

#define NSFPS_OUT8(a, i)                                                                    \
  "=r"(a[i]), "=r"(a[i + 1]), "=r"(a[i + 2]), "=r"(a[i + 3]), "=r"(a[i + 4]), "=r"(a[i + 5]), \
      "=r"(a[i + 6]), "=r"(a[i + 7])
#define NSFPS_IN8(a, i)                                                                  \
  "r"(a[i]), "r"(a[i + 1]), "r"(a[i + 2]), "r"(a[i + 3]), "r"(a[i + 4]), "r"(a[i + 5]),  \
      "r"(a[i + 6]), "r"(a[i + 7])

// 32 consecutive columns of this warp's 32 lanes, one lane each.  The values
// are there after tmem_ld_wait().
__device__ __forceinline__ void tmem_ld32(uint32_t (&r)[32], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : NSFPS_OUT8(r, 0), NSFPS_OUT8(r, 8), NSFPS_OUT8(r, 16), NSFPS_OUT8(r, 24)
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(addr), NSFPS_IN8(r, 0), NSFPS_IN8(r, 8), NSFPS_IN8(r, 16), NSFPS_IN8(r, 24)
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t (&r)[16], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15}, [%16];"
      : NSFPS_OUT8(r, 0), NSFPS_OUT8(r, 8)
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16};" ::"r"(addr), NSFPS_IN8(r, 0), NSFPS_IN8(r, 8)
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr),
               NSFPS_IN8(r, 0)
               : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// A barrier whose phase completes after `count` arrivals (a commit is one).
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count = 1u) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Waits for the phase of parity `phase`; false when it has not come after
// limit_ns (a product that never ends), which no working call sees.
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t phase) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.b32 %0, 1, 0, p;\n}"
      : "=r"(done)
      : "r"(bar), "r"(phase)
      : "memory");
  return done;
}
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t phase,
                                         unsigned long long limit_ns) {
  if (bar_try(bar, phase)) return true;
  unsigned long long begin, now;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(begin));
  do {
    if (bar_try(bar, phase)) return true;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
  } while (now - begin < limit_ns);
  return false;
}

}  // namespace nsfps
