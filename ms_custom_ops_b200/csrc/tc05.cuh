// tcgen05 (5th-generation tensor core) wrappers of libmsco_b200.so: TMEM allocation, matrix instructions with
// operands in shared memory or TMEM, moves between TMEM and registers.
#pragma once

#include <stdint.h>

#include "msco_common.cuh"

namespace msco {

#ifdef __CUDACC__
// one lane of a converged warp
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void tmem_alloc(uint32_t *smem_dst, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(smem_dst)), "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t addr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// arrives on the mbarrier once every matrix instruction that this thread has issued so far is complete
__device__ __forceinline__ void tc_commit_at(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_commit(uint64_t *bar) { tc_commit_at(smem_u32(bar)); }

// Shared-memory matrix descriptor, 128-byte swizzle.  K-major operand: rows of 128 bytes (64 16-bit elements of the
// contraction), 8-row groups 1024 bytes apart (stride); the leading offset is not used.  MN-major operand: 64
// elements of the free dimension per 128-byte row, rows along the contraction, 8-row groups 1024 bytes apart
// (stride), the next 64 elements of the free dimension `leading` bytes on.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t leading = 16) {
  return (uint64_t)((addr & 0x3ffff) >> 4) | ((uint64_t)(leading >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// Instruction descriptor of kind::f16 with float32 accumulators: M x N, A K-major, B K-major or MN-major.
template <bool BF16, int M, int N, bool B_MN>
__host__ __device__ constexpr uint32_t mma_idesc() {
  return (1u << 4) | ((BF16 ? 1u : 0u) << 7) | ((BF16 ? 1u : 0u) << 10) | ((B_MN ? 1u : 0u) << 16) |
         ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// D (TMEM) = A (shared) * B (shared) (+ D); one thread issues
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
      "r"((uint32_t)accumulate)
      : "memory");
}
// D (TMEM) = A (TMEM, 16-bit pairs) * B (shared) (+ D)
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
      "r"((uint32_t)accumulate)
      : "memory");
}

// 32 columns of this warp's 32 TMEM lanes: lane i's row in its 32 registers
#define MSCO_R4(r, i) "=r"((r)[i]), "=r"((r)[(i) + 1]), "=r"((r)[(i) + 2]), "=r"((r)[(i) + 3])
#define MSCO_W4(r, i) "r"((r)[i]), "r"((r)[(i) + 1]), "r"((r)[(i) + 2]), "r"((r)[(i) + 3])
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
      "%30,%31}, [%32];"
      : MSCO_R4(r, 0), MSCO_R4(r, 4), MSCO_R4(r, 8), MSCO_R4(r, 12), MSCO_R4(r, 16), MSCO_R4(r, 20), MSCO_R4(r, 24),
        MSCO_R4(r, 28)
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : MSCO_R4(r, 0), MSCO_R4(r, 4), MSCO_R4(r, 8), MSCO_R4(r, 12)
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
      "%30,%31};" ::MSCO_W4(r, 0),
      MSCO_W4(r, 4), MSCO_W4(r, 8), MSCO_W4(r, 12), MSCO_W4(r, 16), MSCO_W4(r, 20), MSCO_W4(r, 24), MSCO_W4(r, 28),
      "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::MSCO_W4(r, 0),
      MSCO_W4(r, 4), MSCO_W4(r, 8), MSCO_W4(r, 12), "r"(addr)
      : "memory");
}
// Waits for this thread's loads from TMEM.  The registers pass through the statement: nothing that reads them can be
// moved in front of it.
#define MSCO_T4(r, i) "+r"((r)[i]), "+r"((r)[(i) + 1]), "+r"((r)[(i) + 2]), "+r"((r)[(i) + 3])
__device__ __forceinline__ void tmem_wait_ld32(uint32_t *r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : MSCO_T4(r, 0), MSCO_T4(r, 4), MSCO_T4(r, 8), MSCO_T4(r, 12), MSCO_T4(r, 16), MSCO_T4(r, 20), MSCO_T4(r, 24),
                 MSCO_T4(r, 28)
               :
               : "memory");
}
__device__ __forceinline__ void tmem_wait_ld16(uint32_t *r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : MSCO_T4(r, 0), MSCO_T4(r, 4), MSCO_T4(r, 8), MSCO_T4(r, 12)
               :
               : "memory");
}
#undef MSCO_T4
#undef MSCO_R4
#undef MSCO_W4

// two float32 operations per instruction
__device__ __forceinline__ uint64_t pack_f32x2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack_f32x2(uint64_t v, float &a, float &b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// 2^x of two values without the special-function unit: x = n + f with n the nearest integer (by adding and subtracting
// 1.5 * 2^23, whose low bits then hold n) and f in [-1/2, 1/2]; 2^f by the cubic of least relative error there (7.5e-5:
// computed for this by linear programming on a grid), n added to the exponent.  x is held above -126 (a NaN stays one), so what should
// be 0 is 2^-126.
__device__ __forceinline__ void exp2_poly2(uint64_t v, float &a, float &b) {
  float x, y;
  unpack_f32x2(v, x, y);
  asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(x));  // -126
  asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(y));
  v = pack_f32x2(x, y);
  const uint64_t t = add_f32x2(v, pack_f32x2(12582912.f, 12582912.f));
  const uint64_t f = fma_f32x2(add_f32x2(t, pack_f32x2(-12582912.f, -12582912.f)), pack_f32x2(-1.f, -1.f), v);
  uint64_t q = fma_f32x2(f, pack_f32x2(0.05517166852951050f, 0.05517166852951050f),
                         pack_f32x2(0.2426111251115799f, 0.2426111251115799f));
  q = fma_f32x2(q, f, pack_f32x2(0.6932609677314758f, 0.6932609677314758f));
  q = fma_f32x2(q, f, pack_f32x2(0.9999280571937561f, 0.9999280571937561f));
  float tx, ty;
  unpack_f32x2(t, tx, ty);
  unpack_f32x2(q, x, y);
  a = __uint_as_float(__float_as_uint(x) + (__float_as_uint(tx) << 23));
  b = __uint_as_float(__float_as_uint(y) + (__float_as_uint(ty) << 23));
}
#endif  // __CUDACC__

}  // namespace msco
