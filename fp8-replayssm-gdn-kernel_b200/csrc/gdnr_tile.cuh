// Warp-level tile helpers shared by the prompt kernels: ldmatrix / stmatrix forms and the
// swizzled shared-memory rows they read.
#pragma once

#include "gdnr_device.cuh"

namespace gdnr {

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// 2^x, flushing denormal results
__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16 bytes to shared memory, zeros where `bytes` is 0 (the source is not read then)
__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// Byte offset of 16-byte chunk c of row r in a tile of rows of ROWB bytes (a multiple of 128):
// chunk c of a row sits at c ^ (r & 7), so eight rows' equal chunks cover all banks.
template <int ROWB>
__device__ __forceinline__ uint32_t swz(int r, int c) {
  return uint32_t(r) * ROWB + (uint32_t(c ^ (r & 7)) << 4);
}

}  // namespace gdnr
