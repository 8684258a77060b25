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

// d += a b (m16n8k16, bf16).  Not volatile: the compiler may move it between the loads around it.
__device__ __forceinline__ void mma_bf16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_f16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// d = a b: the accumulator begins at zero without being set to it
__device__ __forceinline__ void mma_bf16_first(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ void mma_f16_first(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ void stsm_x4_t(uint32_t addr, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(r0), "r"(r1), "r"(r2),
               "r"(r3)
               : "memory");
}

// Named barriers: wait for `count` threads
__device__ __forceinline__ void bar_sync(int id, int count) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(count) : "memory"); }
// ... and whether any of them has `x`
__device__ __forceinline__ bool bar_or(int id, int count, bool x) {
  int r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %3, 0;\n\tbar.red.or.pred p, %1, %2, q;\n\tselp.b32 %0, 1, 0, p;\n\t}"
               : "=r"(r)
               : "r"(id), "r"(count), "r"(int(x))
               : "memory");
  return r != 0;
}

// Two floats in one register pair: one instruction for both
__device__ __forceinline__ uint64_t pack2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// x[0..1] *= f
__device__ __forceinline__ void scale2(float* x, uint64_t f) {
  const float2 r = unpack2(mul2(pack2(x[0], x[1]), f));
  x[0] = r.x, x[1] = r.y;
}

// two floats to packed bf16 (x in the low half), one conversion
__device__ __forceinline__ uint32_t cvt_bf16x2(float x, float y) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
  return r;
}

// x as the sum of two bf16 (pairs packed): 16 bits of mantissa, an error of 2^-17 of x at most
__device__ __forceinline__ void split_bf16x2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = cvt_bf16x2(x, y);
  const float2 h = bf16x2_to_f2(hi);
  lo = cvt_bf16x2(x - h.x, y - h.y);
}

// as the sum of two f16: 22 bits of mantissa, for values that are not far below one or above 2^15
__device__ __forceinline__ void split_f16x2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = pack_f16x2(x - f.x, y - f.y);
}

// as the sum of three, 24 bits: float32 itself
__device__ __forceinline__ void split3_bf16x2(float x, float y, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  hi = cvt_bf16x2(x, y);
  const float2 h = bf16x2_to_f2(hi);
  const float rx = x - h.x, ry = y - h.y;
  mid = cvt_bf16x2(rx, ry);
  const float2 m = bf16x2_to_f2(mid);
  lo = cvt_bf16x2(rx - m.x, ry - m.y);
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

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// Copies in flight end before their CTA does: waits until the last tiles of a ring, `tiles` in all, have landed (one limit for
// all of them).  Whoever requests tiles calls it before leaving, whether its own waits gave up or only those of the others.
__device__ __forceinline__ void drain(uint64_t* full, uint32_t stages, uint32_t tiles) {
  const uint64_t t = globaltimer_ns();
  for (uint32_t k = tiles > stages ? tiles - stages : 0; k < tiles; ++k)
    while (!mbar_try_wait(smem_addr(&full[k % stages]), (k / stages) & 1) && globaltimer_ns() - t < WAIT_LIMIT_NS) {
    }
}

// Waits of a whole warp; they give up after a second, or when another warp has: then every role leaves its loop.
struct WarpWait {
  uint32_t* err;
  volatile int* abort;
  __device__ __forceinline__ bool operator()(uint64_t* bar, uint32_t parity) const {
    bool ok = mbar_try_wait(smem_addr(bar), parity);
    if (!ok) ok = slow(bar, parity);
    return __all_sync(0xffffffffu, ok);
  }
  __device__ __forceinline__ bool slow(uint64_t* bar, uint32_t parity) const {
    const uint32_t a = smem_addr(bar);
    const uint64_t t0 = globaltimer_ns();
    for (uint32_t it = 1; it < WAIT_LIMIT_ITERS; ++it) {
      if (mbar_try_wait(a, parity)) return true;
      if ((it & 63u) == 0) {
        if (*abort) return false;
        if (globaltimer_ns() - t0 > WAIT_LIMIT_NS) break;
      }
    }
    if (mbar_try_wait(a, parity)) return true;  // the warp itself may have been held up since it last looked
    *abort = 1;
    atomicOr(err, GDNR_DEVERR_WAIT_TIMEOUT);
    return false;
  }
};

}  // namespace gdnr
