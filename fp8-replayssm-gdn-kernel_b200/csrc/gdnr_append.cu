// Per-head RMS norm of queries and keys, rotary positions, and the append of keys and
// values to a paged cache, in one pass (gdnr_qk_norm_rope_append).
//
//   y = x / sqrt(mean(x^2) + eps) * (w + w_off)            (heads with a weight)
//   (y_i, y_j) <- (y_i cos - y_j sin, y_j cos + y_i sin)   j = i + rot/2 (half layout) or
//                                                          i = 2m, j = 2m + 1 (interleaved)
// in float32, rounded once when stored.
#include "gdnr_device.cuh"
#include "gdnr_hybrid.h"

namespace gdnr {

namespace {

constexpr int AP_WARPS = 8;

// One warp per (token, head): bound by memory, every value is read and written once.
// The pair of an element can sit in any lane (rot is any even number), so the
// normalised row goes through the warp's own row of shared memory.
template <int D>
__global__ void __launch_bounds__(AP_WARPS * 32) append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int E = D / 32;  // elements a lane holds: 2, 4 or 8
  __shared__ float rows[AP_WARPS][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = p.Hq + 2 * p.Hk;
  const int64_t item = int64_t(blockIdx.x) * AP_WARPS + warp;
  if (item >= int64_t(p.T) * heads) return;
  const int t = int(item / heads), hd = int(item - int64_t(t) * heads);
  const bool is_q = hd < p.Hq, is_k = !is_q && hd < p.Hq + p.Hk;
  const int h = is_q ? hd : (is_k ? hd - p.Hq : hd - p.Hq - p.Hk);
  const uint16_t* src = is_q ? p.q + int64_t(t) * p.q_st + int64_t(h) * p.q_sh
                             : (is_k ? p.k + int64_t(t) * p.k_st + int64_t(h) * p.k_sh
                                     : p.v + int64_t(t) * p.v_st + int64_t(h) * p.v_sh);
  uint16_t* dst = nullptr;
  if (is_q) {
    dst = p.q_out + int64_t(t) * p.qo_st + int64_t(h) * p.qo_sh;
  } else {
    const int slot = p.slots[int64_t(t) * p.sl_s];
    if (slot < 0) return;  // padding
    const int page = slot / p.page_size, at = slot - page * p.page_size;
    if (page >= p.pages) {
      if (lane == 0) atomicOr(p.err, GDNR_DEVERR_BAD_SLOT);
      return;
    }
    dst = is_k ? p.kc + int64_t(page) * p.kc_sp + int64_t(at) * p.kc_st + int64_t(h) * p.kc_sh
               : p.vc + int64_t(page) * p.vc_sp + int64_t(at) * p.vc_st + int64_t(h) * p.vc_sh;
  }
  uint32_t raw[E / 2];
  if constexpr (E == 8) {
    const uint4 w = *reinterpret_cast<const uint4*>(src + lane * 8);
    raw[0] = w.x, raw[1] = w.y, raw[2] = w.z, raw[3] = w.w;
  } else if constexpr (E == 4) {
    const uint2 w = *reinterpret_cast<const uint2*>(src + lane * 4);
    raw[0] = w.x, raw[1] = w.y;
  } else {
    raw[0] = *reinterpret_cast<const uint32_t*>(src + lane * 2);
  }
  if (is_q || is_k) {
    float x[E];
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const float2 f = bf16x2_to_f2(raw[i]);
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
    const void* w = is_q ? p.qw : p.kw;
    if (w) {
      const int wdt = is_q ? p.qw_dt : p.kw_dt;
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) ss += x[i] * x[i];
      ss = warp_sum(ss);
      const float r = 1.0f / sqrtf(ss * (1.0f / D) + p.eps);
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = x[i] * r * (load_scalar(w, lane * E + i, wdt) + p.w_off);
    }
    const int pos = p.pos[int64_t(t) * p.pos_s];
    if (pos < 0 || pos >= p.P) {  // no angles for it: the head stays unrotated
      if (lane == 0) atomicOr(p.err, GDNR_DEVERR_BAD_POS);
    } else {
      const float* tb = p.table + int64_t(pos) * p.tb_s;
      const int half = p.rot >> 1;
#pragma unroll
      for (int i = 0; i < E; ++i) rows[warp][lane * E + i] = x[i];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int c = lane * E + i;
        if (c < p.rot) {
          const int m = p.inter ? c >> 1 : (c < half ? c : c - half);
          const bool first = p.inter ? !(c & 1) : c < half;
          const int o = p.inter ? c ^ 1 : (first ? c + half : c - half);
          const float cs = tb[m], sn = tb[half + m], y = rows[warp][o];
          x[i] = first ? x[i] * cs - y * sn : x[i] * cs + y * sn;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < E / 2; ++i) raw[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
  }
  if constexpr (E == 8)
    *reinterpret_cast<uint4*>(dst + lane * 8) = make_uint4(raw[0], raw[1], raw[2], raw[3]);
  else if constexpr (E == 4)
    *reinterpret_cast<uint2*>(dst + lane * 4) = make_uint2(raw[0], raw[1]);
  else
    *reinterpret_cast<uint32_t*>(dst + lane * 2) = raw[0];
}

}  // namespace

cudaError_t launch_append(const AppendParams& p, cudaStream_t stream) {
  const int64_t items = int64_t(p.T) * (p.Hq + 2 * p.Hk);
  const dim3 grid(unsigned((items + AP_WARPS - 1) / AP_WARPS));
  if (p.D == 64)
    append_kernel<64><<<grid, AP_WARPS * 32, 0, stream>>>(p);
  else if (p.D == 128)
    append_kernel<128><<<grid, AP_WARPS * 32, 0, stream>>>(p);
  else
    append_kernel<256><<<grid, AP_WARPS * 32, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace gdnr
