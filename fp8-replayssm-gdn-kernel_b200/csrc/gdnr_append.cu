// Per-head RMS norm of queries and keys, rotary positions, and the append of keys and
// values to a paged cache, in one pass (gdnr_qk_norm_rope_append).
//
//   y = x / sqrt(mean(x^2) + eps) * (w + w_off)            (heads with a weight)
//   (y_i, y_j) <- (y_i cos - y_j sin, y_j cos + y_i sin)   j = i + rot/2 (half layout) or
//                                                          i = 2m, j = 2m + 1 (interleaved)
// in float32, rounded once when stored.
#include "gdnr_device.cuh"
#include "gdnr_hybrid.h"
#include "gdnr_tile.cuh"

#include <algorithm>

namespace gdnr {

namespace {

constexpr int AP_WARPS = 8;

// How a lane finds the other element of a rotated pair: it holds both (interleaved); it is in the
// lane half / 8 further or back (half layout, half a multiple of 8); or anywhere, then the head
// goes through shared memory.
enum ApPair { AP_OWN, AP_HOP, AP_ANY };

__device__ __forceinline__ void ap_floats8(const float* src, float* x) {
  const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}

// Bound by memory: every value is read and written once.  A lane has eight neighbouring elements (16
// bytes) of a head, so D / 8 lanes a head and 1, 2 or 4 heads a warp at a time; a warp has ITER such
// sets of one kind (queries, keys or values) and walks `per_warp` tokens with them, the next
// token's rows, position and slot on their way.  Weights are fetched once a warp, angles once a
// token.  Arithmetic on pairs: it is the instructions that cost (8192 tokens of 16 + 2 + 2 heads of
// 256: 98 us with a warp for one head of one token and scalar operations).
template <int D, int ITER, int PAIR>
__global__ void __launch_bounds__(AP_WARPS * 32, 3) append_kernel(const __grid_constant__ AppendParams p, const int per_warp) {
  constexpr int LPH = D / 8, HPI = 32 / LPH, HPW = HPI * ITER;
  __shared__ float rows[PAIR == AP_ANY ? AP_WARPS : 1][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, li = lane & (LPH - 1), c0 = li * 8;
  const uint32_t gq = uint32_t(p.Hq + HPW - 1) / HPW, gk = uint32_t(p.Hk + HPW - 1) / HPW, groups = gq + 2 * gk;
  const uint32_t item = blockIdx.x * AP_WARPS + warp, block = item / groups;
  uint32_t g = item - block * groups;
  if (block * uint32_t(per_warp) >= uint32_t(p.T)) return;
  int t = int(block) * per_warp;
  const int t_end = min(t + per_warp, p.T);
  const bool is_q = g < gq, is_v = g >= gq + gk;
  g -= is_q ? 0 : (is_v ? gq + gk : gq);
  const int h0 = int(g) * HPW + lane / LPH, heads = is_q ? p.Hq : p.Hk;  // the lane's heads: h0 + j HPI
  const int64_t sh = is_q ? p.q_sh : (is_v ? p.v_sh : p.k_sh), st = is_q ? p.q_st : (is_v ? p.v_st : p.k_st);
  const uint16_t* src = (is_q ? p.q : (is_v ? p.v : p.k)) + t * st + h0 * sh + c0;
  uint16_t* const base = (is_q ? p.q_out : (is_v ? p.vc : p.kc)) + c0 + h0 * (is_q ? p.qo_sh : (is_v ? p.vc_sh : p.kc_sh));
  const int64_t dh = is_q ? p.qo_sh : (is_v ? p.vc_sh : p.kc_sh);
  const int64_t d_page = is_v ? p.vc_sp : p.kc_sp, d_row = is_v ? p.vc_st : p.kc_st;
  uint4 next[ITER];
  int next_slot = 0, next_pos = 0;
  auto request = [&](int tt) {
#pragma unroll
    for (int j = 0; j < ITER; ++j) {
      next[j] = make_uint4(0, 0, 0, 0);
      if (h0 + j * HPI < heads) next[j] = *reinterpret_cast<const uint4*>(src + j * HPI * sh);
    }
    src += st;
    if (!is_q) next_slot = p.slots[tt * p.sl_s];
    if (!is_v) next_pos = p.pos[tt * p.pos_s];
  };
  request(t);
  const void* w = is_q ? p.qw : (is_v ? nullptr : p.kw);
  uint64_t wt[4];
  if (w) {  // 16-byte aligned: the host sees to it
    float f[8];
    if ((is_q ? p.qw_dt : p.kw_dt) == GDNR_F32) {
      ap_floats8(static_cast<const float*>(w) + c0, f);
    } else {
      const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(w) + c0);
      const uint32_t vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 y = bf16x2_to_f2(vv[i]);
        f[2 * i] = y.x, f[2 * i + 1] = y.y;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) wt[i] = pack2(f[2 * i] + p.w_off, f[2 * i + 1] + p.w_off);
  }
  const int half = p.rot >> 1;
  const int hop = half / 8, peer = li < hop ? lane + hop : (li < 2 * hop ? lane - hop : lane);
  const float sign = c0 < half ? -1.f : 1.f;
  for (; t < t_end; ++t) {
    uint4 raw[ITER];
#pragma unroll
    for (int j = 0; j < ITER; ++j) raw[j] = next[j];
    const int slot = next_slot, pos = next_pos;
    if (t + 1 < t_end) request(t + 1);
    uint16_t* dst = base;
    if (is_q) {
      dst += t * p.qo_st;
    } else {
      if (slot < 0) continue;  // padding
      const int page = p.page_shift >= 0 ? slot >> p.page_shift : slot / p.page_size;
      if (page >= p.pages) {
        if (lane == 0) atomicOr(p.err, GDNR_DEVERR_BAD_SLOT);
        continue;
      }
      dst += page * d_page + (slot - page * p.page_size) * d_row;
    }
    if (!is_v) {
      const bool rotate = pos >= 0 && pos < p.P;
      if (!rotate && lane == 0) atomicOr(p.err, GDNR_DEVERR_BAD_POS);  // the heads stay unrotated
      // angles of the lane's elements; the sine carries the sign of the pair's other element
      float cs[8], sn[8];
      if (rotate && p.tb_vec && c0 < p.rot) {  // rows of whole 16-byte pieces, half a multiple of 8
        const float* tb = p.table + pos * p.tb_s;
        if constexpr (PAIR == AP_OWN) {
          const float4 a = *reinterpret_cast<const float4*>(tb + li * 4), b = *reinterpret_cast<const float4*>(tb + half + li * 4);
          cs[0] = cs[1] = a.x, cs[2] = cs[3] = a.y, cs[4] = cs[5] = a.z, cs[6] = cs[7] = a.w;
          sn[0] = -b.x, sn[1] = b.x, sn[2] = -b.y, sn[3] = b.y, sn[4] = -b.z, sn[5] = b.z, sn[6] = -b.w, sn[7] = b.w;
        } else {
          const int m = c0 < half ? c0 : c0 - half;
          ap_floats8(tb + m, cs);
          ap_floats8(tb + half + m, sn);
#pragma unroll
          for (int i = 0; i < 8; ++i) sn[i] *= sign;
        }
      } else {
        const float* tb = p.table + int64_t(rotate ? pos : 0) * p.tb_s;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int c = c0 + i;
          cs[i] = 1.f, sn[i] = 0.f;
          if (rotate && c < p.rot) {
            const int m = PAIR == AP_OWN ? c >> 1 : (c < half ? c : c - half);
            cs[i] = tb[m];
            sn[i] = (PAIR == AP_OWN ? !(c & 1) : c < half) ? -tb[half + m] : tb[half + m];
          }
        }
      }
#pragma unroll
      for (int j = 0; j < ITER; ++j) {
        if (int(g) * HPW + j * HPI >= heads) break;  // no head of the set exists
        uint32_t* rw = reinterpret_cast<uint32_t*>(&raw[j]);
        uint64_t x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = bf16x2_to_f2(rw[i]);
          x[i] = pack2(f.x, f.y);
        }
        if (w) {
          uint64_t s2 = mul2(x[0], x[0]);
#pragma unroll
          for (int i = 1; i < 4; ++i) s2 = fma2(x[i], x[i], s2);
          const float2 sp = unpack2(s2);
          float ss = sp.x + sp.y;
#pragma unroll
          for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          const float r = rsqrtf(ss * (1.0f / D) + p.eps);
          const uint64_t r2 = pack2(r, r);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = mul2(mul2(x[i], r2), wt[i]);
        }
        if (rotate) {
          float y[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = unpack2(x[i]);
            y[2 * i] = f.x, y[2 * i + 1] = f.y;
          }
          if constexpr (PAIR == AP_OWN) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float z = y[2 * i];
              y[2 * i] = y[2 * i + 1], y[2 * i + 1] = z;
            }
          } else if constexpr (PAIR == AP_HOP) {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = __shfl_sync(0xffffffffu, y[i], peer);
          } else {
            float* row = rows[warp] + lane / LPH * D;
#pragma unroll
            for (int i = 0; i < 8; ++i) row[c0 + i] = y[i];
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int c = c0 + i;
              y[i] = c < p.rot ? row[c < half ? c + half : c - half] : 0.f;
            }
            __syncwarp();
          }
          if (c0 < p.rot)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint64_t z =
                  fma2(pack2(y[2 * i], y[2 * i + 1]), pack2(sn[2 * i], sn[2 * i + 1]), mul2(x[i], pack2(cs[2 * i], cs[2 * i + 1])));
              if (PAIR == AP_HOP || c0 + 2 * i < p.rot) x[i] = z;  // (rot is even: it ends between pairs)
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = unpack2(x[i]);
          rw[i] = cvt_bf16x2(f.x, f.y);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < ITER; ++j)
      if (h0 + j * HPI < heads) *reinterpret_cast<uint4*>(dst + j * HPI * dh) = raw[j];
  }
}

template <int D, int ITER>
cudaError_t run(const AppendParams& p, int per_warp, cudaStream_t stream) {
  constexpr int HPW = 256 / D * ITER;
  const int64_t groups = (p.Hq + HPW - 1) / HPW + 2 * ((p.Hk + HPW - 1) / HPW);
  const dim3 grid(unsigned(((int64_t(p.T) + per_warp - 1) / per_warp * groups + AP_WARPS - 1) / AP_WARPS));
  if (p.inter)
    append_kernel<D, ITER, AP_OWN><<<grid, AP_WARPS * 32, 0, stream>>>(p, per_warp);
  else if ((p.rot / 2) % 8 == 0)
    append_kernel<D, ITER, AP_HOP><<<grid, AP_WARPS * 32, 0, stream>>>(p, per_warp);
  else
    append_kernel<D, ITER, AP_ANY><<<grid, AP_WARPS * 32, 0, stream>>>(p, per_warp);
  return cudaGetLastError();
}

template <int D>
cudaError_t pick(const AppendParams& p, cudaStream_t stream) {
  // two sets and several tokens a warp where that still fills the machine with warps, else one of one token
  const int64_t bytes = int64_t(p.T) * (p.Hq + 2 * p.Hk) * D * 2, full = int64_t(multiprocessor_count()) * 32 * 1024;
  return bytes >= full ? run<D, 2>(p, int(std::min<int64_t>(4, bytes / full)), stream) : run<D, 1>(p, 1, stream);
}

}  // namespace

cudaError_t launch_append(const AppendParams& p, cudaStream_t stream) {
  if (p.D == 64) return pick<64>(p, stream);
  if (p.D == 128) return pick<128>(p, stream);
  return pick<256>(p, stream);
}

}  // namespace gdnr
