// Fifth-generation tensor core primitives (sm_100a): tensor memory, descriptors, issue and completion.
#pragma once

#include <stdint.h>

#include <type_traits>

namespace mcop {

// Allocates / frees all 512 columns of the SM's tensor memory (whole warp); the address goes to shared memory.
__device__ __forceinline__ void tmem_alloc_all(uint32_t* out_smem) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"((uint32_t)__cvta_generic_to_shared(out_smem)) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free_all(uint32_t addr) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(addr) : "memory");
}

// 32 columns of fp32 of this warp's 32 lanes, one lane per thread.  A load's values may be used after tmem_wait_ld().
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
               "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
                 "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]),
                 "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]),
                 "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
               : "r"(addr));
}
// The same for 8 columns.
__device__ __forceinline__ void tmem_ld8(uint32_t addr, float* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "r"(addr));
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const float* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
               "%16};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
                 "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Keeps the uses of 32 loaded values behind the wait that precedes this call.
__device__ __forceinline__ void tmem_loaded32(float* v) {
  asm volatile(""
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]),
                 "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]),
                 "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]),
                 "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31]));
}
__device__ __forceinline__ void tmem_loaded8(float* v) {
  asm volatile("" : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Order of tensor-memory accesses across a barrier: before an arrive, after a wait.
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// The functions below are called by a whole warp; one elected thread, always the same one, issues.
// The mbarrier gets one arrival when every MMA issued so far is complete.
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
                   (uint32_t)__cvta_generic_to_shared(bar))
               : "memory");
}

// Descriptor of a shared-memory operand in the 128-byte swizzle: rows of 128 bytes, 8 rows to an atom of 1024 bytes, atoms one behind
// the other.  The low word: address, and lbo, the bytes between 64-element blocks of the M / N dimension (operands that are
// contiguous along M / N only).  The high word is the same for all.  Offsets add to the low word in units of 16 bytes.
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, uint32_t lbo) { return (addr & 0x3ffff) >> 4 | (lbo >> 4) << 16; }
constexpr uint32_t kDescHigh = 1024 / 16 | 1u << 14 | 2u << 29;
// Instruction descriptor of kind::f16 with an fp32 accumulator.  bf16: both operands bf16 (otherwise both f16).
__host__ __device__ constexpr uint32_t f16_idesc(bool bf16, int m, int n, bool b_mn_major) {
  return 1u << 4 | (bf16 ? 1u : 0u) << 7 | (bf16 ? 1u : 0u) << 10 | (b_mn_major ? 1u : 0u) << 16 | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}
// D[tmem] (+)= A[smem] B[smem], both operands OFF bytes behind their bases (the additions stay inside: hoisted out of a loop, the
// descriptors of its products would fill the issuing thread's registers)
template <uint32_t IDESC, uint32_t A_OFF, uint32_t B_OFF> __device__ __forceinline__ void tc_mma_ss(uint32_t d, uint32_t a, uint32_t b, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b32 x, y, i;\n\t.reg .b64 da, db;\n\tsetp.ne.u32 p, %3, 0;\n\tadd.u32 x, %1, %4;\n\tadd.u32 y, %2, %5;\n\t"
      "mov.b32 i, %6;\n\tmov.b64 da, {x, %7};\n\tmov.b64 db, {y, %7};\n\t"
      "elect.sync _|e, 0xffffffff;\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, i, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"((uint32_t)accumulate), "n"(A_OFF / 16), "n"(B_OFF / 16),
      "n"(IDESC), "r"(kDescHigh)
      : "memory");
}
// D[tmem] (+)= A[tmem] B[smem]; A_OFF in columns
template <uint32_t IDESC, uint32_t A_OFF, uint32_t B_OFF> __device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint32_t b, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b32 x, y, i;\n\t.reg .b64 db;\n\tsetp.ne.u32 p, %3, 0;\n\tadd.u32 x, %1, %4;\n\tadd.u32 y, %2, %5;\n\t"
      "mov.b32 i, %6;\n\tmov.b64 db, {y, %7};\n\t"
      "elect.sync _|e, 0xffffffff;\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x], db, i, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"((uint32_t)accumulate), "n"(A_OFF), "n"(B_OFF / 16),
      "n"(IDESC), "r"(kDescHigh)
      : "memory");
}
// Runs f(integral_constant<int, 0>), ..., f(integral_constant<int, N - 1>).
template <int N, int I = 0, typename F> __device__ __forceinline__ void static_for(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    static_for<N, I + 1>(f);
  }
}

}  // namespace mcop
