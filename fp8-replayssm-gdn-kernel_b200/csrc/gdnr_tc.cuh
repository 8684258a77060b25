// The fifth-generation tensor cores: descriptors, products, tensor memory.
#pragma once

#include "gdnr_tile.cuh"

namespace gdnr {

// Matrix descriptors, the low words (the start address is added, in units of 16 bytes): 128-byte swizzle, groups of eight rows
// 1024 bytes apart.  Rows of 128 bytes with K along them: the other distance is not used.  Rows of 128 bytes (64
// elements of N) with K across them: column blocks `lbo` bytes apart.
__host__ __device__ constexpr uint32_t tc_low_k() { return 1u << 16; }
__host__ __device__ constexpr uint32_t tc_low_mn(uint32_t lbo) { return (lbo >> 4) << 16; }
constexpr uint32_t TC_HIGH = (1024u >> 4) | (1u << 14) | (2u << 29);
// Rows of 32 bytes with K along them, 32-byte swizzle: groups of eight rows 256 bytes apart.
constexpr uint32_t TC_HIGH_32 = (256u >> 4) | (1u << 14) | (6u << 29);

// One lane of a whole warp.  (With a branch on the lane number instead, the compiler moves every operand of an
// instruction that wants uniform registers there one by one: 58 ns a product against 36.)
__device__ __forceinline__ bool tc_elect() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

// f32 accumulator, bf16 operands (f16 in tc_idesc_f16), M = 128; B with N contiguous where `bn`
__host__ __device__ constexpr uint32_t tc_idesc(int n, bool bn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (bn ? 1u << 16 : 0u) | (uint32_t(n >> 3) << 17) | ((128u >> 4) << 24);
}

__host__ __device__ constexpr uint32_t tc_idesc_f16(int n) { return (1u << 4) | (uint32_t(n >> 3) << 17) | ((128u >> 4) << 24); }

// acc 0: d = a b, else d += a b
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .b64 da, db;\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(TC_HIGH)
      : "memory");
}

template <uint32_t HIGH = TC_HIGH>
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .b64 db;\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(HIGH)
      : "memory");
}

__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

#define TC_R8(o) "=f"(r[o]), "=f"(r[o + 1]), "=f"(r[o + 2]), "=f"(r[o + 3]), "=f"(r[o + 4]), "=f"(r[o + 5]), "=f"(r[o + 6]), "=f"(r[o + 7])
#define TC_W8(o) "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7])

// 32 columns of the thread's lane; the values are there after tc_wait_ld
__device__ __forceinline__ void tc_ld32(uint32_t addr, float* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : TC_R8(0), TC_R8(8), TC_R8(16), TC_R8(24)
      : "r"(addr)
      : "memory");
}

__device__ __forceinline__ void tc_ld16(uint32_t addr, float* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : TC_R8(0), TC_R8(8)
      : "r"(addr)
      : "memory");
}

__device__ __forceinline__ void tc_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::TC_W8(0),
      TC_W8(8), "r"(addr)
      : "memory");
}

__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

}  // namespace gdnr
