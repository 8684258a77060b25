// The gated delta rule over ragged sequences (gdnr_gdn_prefill).
//
//   S_t = e^{g_t} S_{t-1} + d_t k_t^T,   d_t = beta_t (v_t - e^{g_t} S_{t-1} k_t),   o_t = S_t q_t
//
// per value head, S [V, K] float32, with k = k_raw / sqrt(|k_raw|^2 + eps), q likewise times
// K^-1/2, g = -exp(A_log) softplus(a + dt_bias), beta = sigmoid(b).
#include "gdnr_device.cuh"
#include "gdnr_hybrid.h"
#include "gdnr_tile.cuh"

namespace gdnr {

namespace {

// log(1 + e^x), x itself above the threshold the gates of the decode step use.
__device__ __forceinline__ float softplus_gate(float x) { return x > SOFTPLUS_THRESHOLD ? x : log1pf(expf(x)); }

__device__ __forceinline__ float sigmoid_f(float x) { return 1.0f / (1.0f + expf(-x)); }

// ---------------------------------------------------------------- recurrent form
// One warp owns 8 value rows of S in registers (lane: 4 key columns of each), a CTA 32
// rows, so a head is four CTAs and a batch of single tokens reads and writes each state
// once, in 512-byte row pieces.  S k and S q are both taken from the state before the
// update (o = e^g S q + d (k.q)), so a token has one chain of shuffles.  The sums of 8 rows
// over 32 lanes are folded together: 4 + 2 + 1 exchanges halve the rows a lane holds,
// 2 more finish the sum, 9 shuffles instead of 40.
constexpr int RC_ROWS = 8;
constexpr int RC_WARPS = 4;

// Sum over the warp of x[r], r = 0..7; lane l gets row (l >> 2).
__device__ __forceinline__ float fold8(const float* x, int lane) {
  const unsigned full = 0xffffffffu;
  float y[4], z[2];
  const bool h16 = lane & 16, h8 = lane & 8, h4 = lane & 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float keep = h16 ? x[4 + i] : x[i], give = h16 ? x[i] : x[4 + i];
    y[i] = keep + __shfl_xor_sync(full, give, 16);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float keep = h8 ? y[2 + i] : y[i], give = h8 ? y[i] : y[2 + i];
    z[i] = keep + __shfl_xor_sync(full, give, 8);
  }
  float s = (h4 ? z[1] : z[0]) + __shfl_xor_sync(full, h4 ? z[0] : z[1], 4);
  s += __shfl_xor_sync(full, s, 2);
  s += __shfl_xor_sync(full, s, 1);
  return s;
}

struct RcToken {
  uint2 q, k;
  uint16_t v;
  float a, b;
};

__device__ __forceinline__ RcToken rc_load(const PrefillParams& p, int t, int h, int hv, int row, int lane) {
  RcToken x;
  const uint16_t* m = p.mixed + int64_t(t) * p.mx_s;
  x.q = *reinterpret_cast<const uint2*>(m + h * 128 + lane * 4);
  x.k = *reinterpret_cast<const uint2*>(m + (p.H + h) * 128 + lane * 4);
  x.v = m[(2 * p.H + hv) * 128 + row];
  x.a = load_scalar(p.a, int64_t(t) * p.a_st + int64_t(hv) * p.a_sh, p.a_dt);
  x.b = load_scalar(p.b, int64_t(t) * p.b_st + int64_t(hv) * p.b_sh, p.b_dt);
  return x;
}

__global__ void __launch_bounds__(RC_WARPS * 32) prefill_recurrent_kernel(const __grid_constant__ PrefillParams p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int PARTS = 128 / (RC_ROWS * RC_WARPS);
  const int part = blockIdx.x % PARTS, nh = blockIdx.x / PARTS;
  const int n = nh / p.HV, hv = nh - n * p.HV, h = hv / (p.HV / p.H);
  const int row0 = part * (RC_ROWS * RC_WARPS) + warp * RC_ROWS;
  const int my_row = row0 + (lane >> 2);
  const SeqRange r = prefill_seq(p, n);
  if (r.slot < 0) {
    if ((lane & 3) == 0)
      for (int t = r.begin; t < r.end; ++t) p.out[int64_t(t) * p.o_st + int64_t(hv) * p.o_sh + my_row] = 0;
    return;
  }
  const bool fresh = p.has_init && !p.has_init[n * p.hi_s];
  if (r.begin == r.end && !fresh) return;
  float* st = p.state + int64_t(r.slot) * p.st_ss + int64_t(hv) * p.st_sh + int64_t(row0) * 128 + lane * 4;
  float4 S[RC_ROWS];
#pragma unroll
  for (int i = 0; i < RC_ROWS; ++i)
    S[i] = fresh ? make_float4(0.f, 0.f, 0.f, 0.f) : *reinterpret_cast<const float4*>(st + i * 128);
  const float neg_a = -expf(p.a_log[hv * p.al_s]), dtb = p.dt_bias[hv * p.db_s];
  RcToken nx = {};
  if (r.begin < r.end) nx = rc_load(p, r.begin, h, hv, my_row, lane);
  for (int t = r.begin; t < r.end; ++t) {
    const RcToken x = nx;
    if (t + 1 < r.end) nx = rc_load(p, t + 1, h, hv, my_row, lane);
    const float2 q01 = bf16x2_to_f2(x.q.x), q23 = bf16x2_to_f2(x.q.y), k01 = bf16x2_to_f2(x.k.x), k23 = bf16x2_to_f2(x.k.y);
    float qq = q01.x * q01.x + q01.y * q01.y + q23.x * q23.x + q23.y * q23.y;
    float kk = k01.x * k01.x + k01.y * k01.y + k23.x * k23.x + k23.y * k23.y;
    float qk = q01.x * k01.x + q01.y * k01.y + q23.x * k23.x + q23.y * k23.y;
    float sk[RC_ROWS], sq[RC_ROWS];
#pragma unroll
    for (int i = 0; i < RC_ROWS; ++i) {
      sk[i] = S[i].x * k01.x + S[i].y * k01.y + S[i].z * k23.x + S[i].w * k23.y;
      sq[i] = S[i].x * q01.x + S[i].y * q01.y + S[i].z * q23.x + S[i].w * q23.y;
    }
    const float g = neg_a * softplus_gate(x.a + dtb), alpha = expf(g), beta = sigmoid_f(x.b);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      qq += __shfl_xor_sync(0xffffffffu, qq, o);
      kk += __shfl_xor_sync(0xffffffffu, kk, o);
      qk += __shfl_xor_sync(0xffffffffu, qk, o);
    }
    const float rk = 1.0f / sqrtf(kk + L2_EPS), rq = 0.08838834764831845f / sqrtf(qq + L2_EPS);
    const float my_sk = fold8(sk, lane) * rk, my_sq = fold8(sq, lane) * rq;
    const float d = beta * (bf16_to_f(x.v) - alpha * my_sk);
    if ((lane & 3) == 0)
      p.out[int64_t(t) * p.o_st + int64_t(hv) * p.o_sh + my_row] = f_to_bf16(alpha * my_sq + d * (qk * rk * rq));
    const float dk = d * rk;
#pragma unroll
    for (int i = 0; i < RC_ROWS; ++i) {
      const float di = __shfl_sync(0xffffffffu, dk, i * 4);
      S[i].x = alpha * S[i].x + di * k01.x;
      S[i].y = alpha * S[i].y + di * k01.y;
      S[i].z = alpha * S[i].z + di * k23.x;
      S[i].w = alpha * S[i].w + di * k23.y;
    }
  }
#pragma unroll
  for (int i = 0; i < RC_ROWS; ++i) *reinterpret_cast<float4*>(st + i * 128) = S[i];
}

// ---------------------------------------------------------------- chunked form
// Chunks of C = 64 tokens.  With G_i the sum of the gates up to token i of the chunk, raw rows
// K, Q, V and their inverse norms rk, rq:
//   X = S K^T,                       R = beta (V^T - e^G rk X)
//   N = R T^T,    T = (I + A)^-1,    A_ij = beta_i rk_i rk_j e^{G_i - G_j} k_i.k_j      (j < i)
//   O = e^G rq S Q^T + N P^T,        P_ij = rq_i rk_j e^{G_i - G_j} q_i.k_j             (j <= i)
//   S = e^{G_C} S + N diag(e^{G_C - G_j} rk_j) K
// (N [V, C] holds the tokens' new values).  All with value rows as the rows of the matrix
// products, so a warp that owns 16 value rows of S keeps S, X, R and N in registers: the
// accumulators of one product are the left operand of the next, and nothing of the chain
// from one state to the next passes through shared memory or waits for another warp.
//
// A CTA has 64 value rows of a head: four consumer warps of 16 rows and four producer warps
// that load the next chunk and derive T and P of the chunk after the one being consumed.
//
// Rounding: K, Q, V are bf16 as they come.  S, R, T, N and P meet the tensor cores as sums of
// two bf16 (three products where both sides are split), the weighted N as a sum of three (its
// products add up in S, which may be far smaller than their sum of sizes); this keeps the
// float32 state within 1e-5 also where keys are alike.  The output needs it too, although it is bf16: where keys are alike, S Q^T and N P^T
// nearly cancel, and operands rounded once left it 8e-3 off instead of 2e-3.
// Gates are summed in double: differences of float32 prefix sums would cancel under
// strong decay.
constexpr int CK_C = 64;
constexpr int CK_ROWS = 64;
constexpr int CK_THREADS = 256;
constexpr int CK_LDA = 68;  // floats of a row of A and T in float32

struct CkTile {  // one chunk's raw rows, 16-byte chunks swizzled
  uint8_t k[CK_C * 256], q[CK_C * 256], v[CK_C * CK_ROWS * 2];
};
struct CkDerived {
  uint8_t t_hi[CK_C * 128], t_lo[CK_C * 128], p_hi[CK_C * 128], p_lo[CK_C * 128];
  float beta[CK_C], cx[CK_C], cq[CK_C], cs[CK_C], total;  // beta, beta e^G rk, e^G rq K^-1/2, e^{G_C - G} rk; e^{G_C}
  float pad[15];
};
struct CkSmem {
  CkTile tile[3];
  CkDerived der[2];
  // A below the diagonal blocks; T's diagonal blocks in their place, its block (i, j) in block (j, i)
  float a[CK_C * CK_LDA], y[CK_C * 20];
  uint8_t stage[4][CK_C * 48];
  double g[CK_C];
  float rk[CK_C], rq[CK_C], gbeta[CK_C];
};
static_assert(sizeof(CkSmem) + 1024 <= MAX_DYN_SMEM, "one CTA per SM");

enum { CK_BAR_PROD = 1, CK_BAR_FULL = 2, CK_BAR_EMPTY = 4 };

__device__ __forceinline__ void ck_load(const PrefillParams& p, CkTile& tl, const SeqRange& r, int c, int h, int hv, int v0, int tid) {
  const uint32_t ks = smem_addr(tl.k), qs = smem_addr(tl.q), vs = smem_addr(tl.v);
  const int t0 = r.begin + c * CK_C;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = (tid >> 4) + i * 8, ch = tid & 15;
    const bool ok = t0 + row < r.end;
    const uint16_t* m = p.mixed + int64_t(ok ? t0 + row : r.begin) * p.mx_s + ch * 8;
    cp_async16_zfill(qs + swz<256>(row, ch), m + h * 128, ok ? 16 : 0);
    cp_async16_zfill(ks + swz<256>(row, ch), m + (p.H + h) * 128, ok ? 16 : 0);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = (tid >> 3) + i * 16, ch = tid & 7;
    const bool ok = t0 + row < r.end;
    cp_async16_zfill(vs + swz<128>(row, ch), p.mixed + int64_t(ok ? t0 + row : r.begin) * p.mx_s + (2 * p.H + hv) * 128 + v0 + ch * 8,
                     ok ? 16 : 0);
  }
  cp_async_commit();
}

// Four columns c..c+3 of row r of the 16 x 16 product L R (rows of both CK_LDA or ld floats apart).
__device__ __forceinline__ void ck_mul16(const float* l, const float* rm, int ldr, float* acc) {
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const float x = l[k];
    const float4 y = *reinterpret_cast<const float4*>(rm + k * ldr);
    acc[0] += x * y.x;
    acc[1] += x * y.y;
    acc[2] += x * y.z;
    acc[3] += x * y.w;
  }
}

__device__ void ck_producer(const PrefillParams& p, CkSmem& sm, const SeqRange& r, int h, int hv, int v0, int chunks) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const float neg_a = -expf(p.a_log[hv * p.al_s]), dtb = p.dt_bias[hv * p.db_s];
  ck_load(p, sm.tile[0], r, 0, h, hv, v0, tid);
  auto gate_in = [&](int c, float& a, float& b) {
    const int t = r.begin + c * CK_C + tid;
    a = b = 0.f;
    if (tid < CK_C && c < chunks && t < r.end) {
      a = load_scalar(p.a, int64_t(t) * p.a_st + int64_t(hv) * p.a_sh, p.a_dt);
      b = load_scalar(p.b, int64_t(t) * p.b_st + int64_t(hv) * p.b_sh, p.b_dt);
    }
  };
  float na, nb;
  gate_in(0, na, nb);
  for (int c = 0; c < chunks; ++c) {
    CkTile& tl = sm.tile[c % 3];
    CkDerived& dv = sm.der[c & 1];
    if (c >= 2) bar_sync(CK_BAR_EMPTY + (c & 1), CK_THREADS);  // the consumers are done with chunk c - 2
    const float a = na, b = nb;
    if (c + 1 < chunks)
      ck_load(p, sm.tile[(c + 1) % 3], r, c + 1, h, hv, v0, tid);
    else
      cp_async_commit();
    gate_in(c + 1, na, nb);
    // gates; tokens past the end neither decay nor write
    if (tid < CK_C) {
      const bool in = r.begin + c * CK_C + tid < r.end;
      sm.g[tid] = in ? double(neg_a * softplus_gate(a + dtb)) : 0.0;
      sm.gbeta[tid] = in ? sigmoid_f(b) : 0.f;
    }
    cp_async_wait<1>();
    bar_sync(CK_BAR_PROD, 128);
    if (warp == 0) {
      double x0 = sm.g[2 * lane], x1 = x0 + sm.g[2 * lane + 1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, x1, o);
        if (lane >= o) x0 += y, x1 += y;
      }
      sm.g[2 * lane] = x0;
      sm.g[2 * lane + 1] = x1;
    }
    {
      // inverse norms: thread t has row t & 63 of K or Q
      const int row = tid & 63;
      const uint8_t* base = tid < CK_C ? tl.k : tl.q;
      float ss = 0.f;
#pragma unroll
      for (int ch = 0; ch < 16; ++ch) {
        const uint4 w = *reinterpret_cast<const uint4*>(base + swz<256>(row, ch));
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = bf16x2_to_f2(ww[i]);
          ss += f.x * f.x + f.y * f.y;
        }
      }
      (tid < CK_C ? sm.rk : sm.rq)[row] = (tid < CK_C ? 1.0f : 0.08838834764831845f) / sqrtf(ss + L2_EPS);
    }
    // rows 16 warp .. + 15 of K K^T and Q K^T, up to the diagonal
    float kk[8][4], qk[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) kk[j][e] = qk[j][e] = 0.f;
    const uint32_t ks = smem_addr(tl.k), qs = smem_addr(tl.q);
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      uint32_t ak[4], aq[4];
      ldsm_x4(ks + swz<256>(warp * 16 + (lane & 15), s * 2 + (lane >> 4)), ak);
      ldsm_x4(qs + swz<256>(warp * 16 + (lane & 15), s * 2 + (lane >> 4)), aq);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j > warp) break;
        uint32_t bb[4];
        ldsm_x4(ks + swz<256>(j * 16 + ((lane >> 4) << 3) + (lane & 7), s * 2 + ((lane >> 3) & 1)), bb);
        mma16816_bf16(kk[2 * j], ak, bb[0], bb[1]);
        mma16816_bf16(kk[2 * j + 1], ak, bb[2], bb[3]);
        mma16816_bf16(qk[2 * j], aq, bb[0], bb[1]);
        mma16816_bf16(qk[2 * j + 1], aq, bb[2], bb[3]);
      }
    }
    bar_sync(CK_BAR_PROD, 128);  // prefix sums and norms are in shared memory
    if (tid < CK_C) {
      const double gi = sm.g[tid], gc = sm.g[CK_C - 1];
      const float e = expf(float(gi)), be = sm.gbeta[tid];
      dv.beta[tid] = be;
      dv.cx[tid] = be * e * sm.rk[tid];
      dv.cq[tid] = e * sm.rq[tid];
      dv.cs[tid] = expf(float(gc - gi)) * sm.rk[tid];
      if (tid == 0) dv.total = expf(float(gc));
    }
    {
      const int i0 = warp * 16 + (lane >> 2);
      const double gi[2] = {sm.g[i0], sm.g[i0 + 8]};
      const float bk[2] = {sm.gbeta[i0] * sm.rk[i0], sm.gbeta[i0 + 8] * sm.rk[i0 + 8]}, rq[2] = {sm.rq[i0], sm.rq[i0 + 8]};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j > 2 * warp + 1) break;
        const int col = j * 8 + 2 * (lane & 3);
        const double gj[2] = {sm.g[col], sm.g[col + 1]};
        const float rk[2] = {sm.rk[col], sm.rk[col + 1]};
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          float av[2], pv[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = i0 + 8 * hf;
            const float d = ex2_approx(float(gi[hf] - gj[e]) * 1.4426950408889634f) * rk[e];
            av[e] = col + e < row ? bk[hf] * d * kk[j][2 * hf + e] : 0.f;
            pv[e] = col + e <= row ? rq[hf] * d * qk[j][2 * hf + e] : 0.f;
          }
          const int row = i0 + 8 * hf;
          *reinterpret_cast<float2*>(&sm.a[row * CK_LDA + col]) = make_float2(av[0], av[1]);
          uint32_t ph, pl;
          split_bf16x2(pv[0], pv[1], ph, pl);
          *reinterpret_cast<uint32_t*>(dv.p_hi + swz<128>(row, j) + 4 * (lane & 3)) = ph;
          *reinterpret_cast<uint32_t*>(dv.p_lo + swz<128>(row, j) + 4 * (lane & 3)) = pl;
        }
      }
    }
    __syncwarp();
    // T = (I + A)^-1 by blocks of 16: the warp's diagonal block by substitution, lane = column
    {
      float x[16];
      float* ad = sm.a + (warp * 16) * CK_LDA + warp * 16;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float s0 = i == lane ? 1.f : 0.f, s1 = 0.f;
#pragma unroll
        for (int j = 0; j < i; ++j) {
          if (j & 1)
            s1 -= ad[i * CK_LDA + j] * x[j];
          else
            s0 -= ad[i * CK_LDA + j] * x[j];
        }
        x[i] = s0 + s1;
      }
      __syncwarp();
      if (lane < 16)
#pragma unroll
        for (int i = 0; i < 16; ++i) ad[i * CK_LDA + lane] = x[i];
    }
    bar_sync(CK_BAR_PROD, 128);
    // block (i, j) below: -T_ii (sum over k of A_ik T_kj), one diagonal after the other
#pragma unroll
    for (int d = 1; d < 4; ++d) {
      // 64 groups of (row, four columns) a block
      const int blocks = 4 - d;
      for (int u = tid; u < blocks * 64; u += 128) {
        const int bj = u >> 6, bi = bj + d, rr = (u >> 2) & 15, cc = (u & 3) * 4;
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        for (int k = bj; k < bi; ++k)
          ck_mul16(sm.a + (bi * 16 + rr) * CK_LDA + k * 16, sm.a + (bj * 16) * CK_LDA + k * 16 + cc, CK_LDA, acc);
        *reinterpret_cast<float4*>(&sm.y[(bj * 16 + rr) * 20 + cc]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      }
      bar_sync(CK_BAR_PROD, 128);
      for (int u = tid; u < blocks * 64; u += 128) {
        const int bj = u >> 6, bi = bj + d, rr = (u >> 2) & 15, cc = (u & 3) * 4;
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        ck_mul16(sm.a + (bi * 16 + rr) * CK_LDA + bi * 16, sm.y + (bj * 16) * 20 + cc, 20, acc);
        *reinterpret_cast<float4*>(&sm.a[(bj * 16 + rr) * CK_LDA + bi * 16 + cc]) =
            make_float4(-acc[0], -acc[1], -acc[2], -acc[3]);
      }
      bar_sync(CK_BAR_PROD, 128);
    }
    // T as two bf16: thread t has half a row (what lies right of the diagonal block is never read)
    {
      const int row = tid >> 1, c0 = (tid & 1) * 4;
#pragma unroll
      for (int ch = 0; ch < 4; ++ch) {
        if (c0 + ch > (row >> 4) * 2 + 1) break;
        const int bi = row >> 4, bj = (c0 + ch) >> 1;
        const float* src = sm.a + (bj * 16 + (row & 15)) * CK_LDA + bi * 16 + ((c0 + ch) & 1) * 8;
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) split_bf16x2(src[2 * i], src[2 * i + 1], hi[i], lo[i]);
        *reinterpret_cast<uint4*>(dv.t_hi + swz<128>(row, c0 + ch)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(dv.t_lo + swz<128>(row, c0 + ch)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    }
    bar_arrive(CK_BAR_FULL + (c & 1), CK_THREADS);
  }
}

__device__ void ck_consumer(const PrefillParams& p, CkSmem& sm, const SeqRange& r, int hv, int v0, int chunks, bool fresh) {
  const int warp = (threadIdx.x >> 5) - 4, lane = threadIdx.x & 31;
  const int g = lane >> 2, t2 = 2 * (lane & 3);
  // S as accumulators: tile n has rows g, g + 8 of the warp's 16 and key columns 8n + t2, + 1
  float* st = p.state + int64_t(r.slot) * p.st_ss + int64_t(hv) * p.st_sh + int64_t(v0 + warp * 16 + g) * 128 + t2;
  float S[16][4];
#pragma unroll
  for (int n = 0; n < 16; ++n) {
    float2 x = make_float2(0.f, 0.f), y = x;
    if (!fresh) {
      x = *reinterpret_cast<const float2*>(st + n * 8);
      y = *reinterpret_cast<const float2*>(st + 8 * 128 + n * 8);
    }
    S[n][0] = x.x, S[n][1] = x.y, S[n][2] = y.x, S[n][3] = y.y;
  }
  const uint32_t stage = smem_addr(sm.stage[warp]);
  for (int c = 0; c < chunks; ++c) {
    const CkTile& tl = sm.tile[c % 3];
    const CkDerived& dv = sm.der[c & 1];
    const uint32_t ks = smem_addr(tl.k), qs = smem_addr(tl.q), vs = smem_addr(tl.v);
    const uint32_t th = smem_addr(dv.t_hi), tlo = smem_addr(dv.t_lo), ph = smem_addr(dv.p_hi),
                   pl = smem_addr(dv.p_lo);
    bar_sync(CK_BAR_FULL + (c & 1), CK_THREADS);
    float X[8][4], O[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) X[j][e] = O[j][e] = 0.f;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      uint32_t hi[4], lo[4];
      split_bf16x2(S[2 * s][0], S[2 * s][1], hi[0], lo[0]);
      split_bf16x2(S[2 * s][2], S[2 * s][3], hi[1], lo[1]);
      split_bf16x2(S[2 * s + 1][0], S[2 * s + 1][1], hi[2], lo[2]);
      split_bf16x2(S[2 * s + 1][2], S[2 * s + 1][3], hi[3], lo[3]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t b[4];
        const uint32_t off = swz<256>(j * 16 + ((lane >> 4) << 3) + (lane & 7), s * 2 + ((lane >> 3) & 1));
        ldsm_x4(ks + off, b);
        mma16816_bf16(X[2 * j], hi, b[0], b[1]);
        mma16816_bf16(X[2 * j + 1], hi, b[2], b[3]);
        mma16816_bf16(X[2 * j], lo, b[0], b[1]);
        mma16816_bf16(X[2 * j + 1], lo, b[2], b[3]);
        ldsm_x4(qs + off, b);
        mma16816_bf16(O[2 * j], hi, b[0], b[1]);
        mma16816_bf16(O[2 * j + 1], hi, b[2], b[3]);
        mma16816_bf16(O[2 * j], lo, b[0], b[1]);
        mma16816_bf16(O[2 * j + 1], lo, b[2], b[3]);
      }
    }
    // R = beta V^T - (beta e^G rk) X, and its halves as the left operand
    uint32_t rh[4][4], rl[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t w[4];  // tokens 16j + t2 (+1), rows g and g + 8; tokens 16j + 8 + t2
      ldsm_x4_t(vs + swz<128>(j * 16 + ((lane >> 4) << 3) + (lane & 7), warp * 2 + ((lane >> 3) & 1)), w);
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int tok = j * 16 + hf * 8 + t2;
        const float2 be = *reinterpret_cast<const float2*>(&dv.beta[tok]), cx = *reinterpret_cast<const float2*>(&dv.cx[tok]),
                     cq = *reinterpret_cast<const float2*>(&dv.cq[tok]);
        const float2 v0f = bf16x2_to_f2(w[2 * hf]), v1f = bf16x2_to_f2(w[2 * hf + 1]);
        float* x = X[2 * j + hf];
        float* o = O[2 * j + hf];
        split_bf16x2(be.x * v0f.x - cx.x * x[0], be.y * v0f.y - cx.y * x[1], rh[j][2 * hf], rl[j][2 * hf]);
        split_bf16x2(be.x * v1f.x - cx.x * x[2], be.y * v1f.y - cx.y * x[3], rh[j][2 * hf + 1], rl[j][2 * hf + 1]);
        o[0] *= cq.x, o[1] *= cq.y, o[2] *= cq.x, o[3] *= cq.y;
      }
    }
    float N[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) N[j][e] = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = j; i < 4; ++i) {
        uint32_t b[4], bl[4];
        const uint32_t off = swz<128>(i * 16 + ((lane >> 4) << 3) + (lane & 7), j * 2 + ((lane >> 3) & 1));
        ldsm_x4(th + off, b);
        ldsm_x4(tlo + off, bl);
        mma16816_bf16(N[2 * i], rh[j], b[0], b[1]);
        mma16816_bf16(N[2 * i + 1], rh[j], b[2], b[3]);
        mma16816_bf16(N[2 * i], rl[j], b[0], b[1]);
        mma16816_bf16(N[2 * i + 1], rl[j], b[2], b[3]);
        mma16816_bf16(N[2 * i], rh[j], bl[0], bl[1]);
        mma16816_bf16(N[2 * i + 1], rh[j], bl[2], bl[3]);
      }
    // the state first: the next chunk waits for it
    uint32_t nh[4][4], nl[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      split_bf16x2(N[2 * j][0], N[2 * j][1], nh[j][0], nl[j][0]);
      split_bf16x2(N[2 * j][2], N[2 * j][3], nh[j][1], nl[j][1]);
      split_bf16x2(N[2 * j + 1][0], N[2 * j + 1][1], nh[j][2], nl[j][2]);
      split_bf16x2(N[2 * j + 1][2], N[2 * j + 1][3], nh[j][3], nl[j][3]);
    }
    const float total = dv.total;
#pragma unroll
    for (int n = 0; n < 16; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) S[n][e] *= total;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t hi[4], lo[4], rest[4];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const float2 cs = *reinterpret_cast<const float2*>(&dv.cs[j * 16 + hf * 8 + t2]);
        const float* x = N[2 * j + hf];
        split3_bf16x2(x[0] * cs.x, x[1] * cs.y, hi[2 * hf], lo[2 * hf], rest[2 * hf]);
        split3_bf16x2(x[2] * cs.x, x[3] * cs.y, hi[2 * hf + 1], lo[2 * hf + 1], rest[2 * hf + 1]);
      }
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        uint32_t b[4];
        ldsm_x4_t(ks + swz<256>(j * 16 + (lane & 15), n * 2 + (lane >> 4)), b);
        mma16816_bf16(S[2 * n], hi, b[0], b[1]);
        mma16816_bf16(S[2 * n + 1], hi, b[2], b[3]);
        mma16816_bf16(S[2 * n], lo, b[0], b[1]);
        mma16816_bf16(S[2 * n + 1], lo, b[2], b[3]);
        mma16816_bf16(S[2 * n], rest, b[0], b[1]);
        mma16816_bf16(S[2 * n + 1], rest, b[2], b[3]);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = j; i < 4; ++i) {
        uint32_t b[4], bl[4];
        const uint32_t off = swz<128>(i * 16 + ((lane >> 4) << 3) + (lane & 7), j * 2 + ((lane >> 3) & 1));
        ldsm_x4(ph + off, b);
        ldsm_x4(pl + off, bl);
        mma16816_bf16(O[2 * i], nh[j], b[0], b[1]);
        mma16816_bf16(O[2 * i + 1], nh[j], b[2], b[3]);
        mma16816_bf16(O[2 * i], nl[j], b[0], b[1]);
        mma16816_bf16(O[2 * i + 1], nl[j], b[2], b[3]);
        mma16816_bf16(O[2 * i], nh[j], bl[0], bl[1]);
        mma16816_bf16(O[2 * i + 1], nh[j], bl[2], bl[3]);
      }
    if (c + 2 < chunks) bar_arrive(CK_BAR_EMPTY + (c & 1), CK_THREADS);
    // O^T to token rows through the warp's own staging rows (48 bytes apart: no bank twice)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      stsm_x4_t(stage + (j * 16 + ((lane >> 4) << 3) + (lane & 7)) * 48 + ((lane >> 3) & 1) * 16, pack_bf16x2(O[2 * j][0], O[2 * j][1]),
                pack_bf16x2(O[2 * j][2], O[2 * j][3]), pack_bf16x2(O[2 * j + 1][0], O[2 * j + 1][1]),
                pack_bf16x2(O[2 * j + 1][2], O[2 * j + 1][3]));
    __syncwarp();
    const int t0 = r.begin + c * CK_C;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = i * 16 + (lane >> 1);
      if (t0 + row < r.end)
        *reinterpret_cast<uint4*>(p.out + int64_t(t0 + row) * p.o_st + int64_t(hv) * p.o_sh + v0 + warp * 16 + (lane & 1) * 8) =
            *reinterpret_cast<const uint4*>(sm.stage[warp] + row * 48 + (lane & 1) * 16);
    }
    __syncwarp();
  }
#pragma unroll
  for (int n = 0; n < 16; ++n) {
    *reinterpret_cast<float2*>(st + n * 8) = make_float2(S[n][0], S[n][1]);
    *reinterpret_cast<float2*>(st + 8 * 128 + n * 8) = make_float2(S[n][2], S[n][3]);
  }
}

// The n-th sequence from the longest down, so that no long one starts last.  One
// warp; batches above 256 sequences keep their order (the count grows with N^2).
__device__ int ck_by_length(const PrefillParams& p, int want, int lane) {
  if (p.N > 256) return want;
  int found = 0;
  for (int n0 = 0; n0 < p.N; n0 += 32) {
    const int n = n0 + lane;
    int rank = -1;
    if (n < p.N) {
      const int len = p.cu[n + 1] - p.cu[n];
      rank = 0;
      for (int m = 0; m < p.N; ++m) {
        const int other = p.cu[m + 1] - p.cu[m];
        rank += other > len || (other == len && m < n);
      }
    }
    const unsigned hit = __ballot_sync(0xffffffffu, rank == want);
    if (hit) found = n0 + __ffs(hit) - 1;
  }
  return found;
}

__global__ void __launch_bounds__(CK_THREADS, 1) prefill_chunk_kernel(const __grid_constant__ PrefillParams p) {
  extern __shared__ uint8_t raw[];
  CkSmem& sm = *reinterpret_cast<CkSmem*>(raw + (-smem_addr(raw) & 1023u));
  const int heads = p.HV * (128 / CK_ROWS);
  const int n = ck_by_length(p, blockIdx.x / heads, threadIdx.x & 31);
  const int part = blockIdx.x % heads, hv = part / (128 / CK_ROWS), v0 = (part % (128 / CK_ROWS)) * CK_ROWS;
  const SeqRange r = prefill_seq(p, n);
  if (r.slot < 0) {  // null slot: zero rows
    for (int i = threadIdx.x; i < (r.end - r.begin) * CK_ROWS; i += CK_THREADS)
      p.out[int64_t(r.begin + i / CK_ROWS) * p.o_st + int64_t(hv) * p.o_sh + v0 + i % CK_ROWS] = 0;
    return;
  }
  const bool fresh = p.has_init && !p.has_init[n * p.hi_s];
  if (r.begin == r.end && !fresh) return;
  const int chunks = (r.end - r.begin + CK_C - 1) / CK_C;
  if (threadIdx.x < 128) {
    if (chunks) ck_producer(p, sm, r, hv / (p.HV / p.H), hv, v0, chunks);
  } else {
    ck_consumer(p, sm, r, hv, v0, chunks, fresh);
  }
}

}  // namespace

cudaError_t launch_prefill_chunk(const PrefillParams& p, cudaStream_t stream) {
  static DynSmemCache cache;
  constexpr int bytes = sizeof(CkSmem) + 1024;
  cudaError_t e = ensure_dyn_smem(reinterpret_cast<const void*>(prefill_chunk_kernel), bytes, cache);
  if (e != cudaSuccess) return e;
  const int64_t blocks = int64_t(p.N) * p.HV * (128 / CK_ROWS);
  prefill_chunk_kernel<<<dim3(unsigned(blocks)), CK_THREADS, bytes, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_prefill(const PrefillParams& p, int max_seqlen, cudaStream_t stream) {
  // The longest sequence as the host knows it, or the mean length
  const int longest = max_seqlen > 0 ? max_seqlen : p.T / p.N + (p.T % p.N != 0);
  return longest <= 8 ? launch_prefill_recurrent(p, stream) : launch_prefill_chunk(p, stream);
}

cudaError_t launch_prefill_recurrent(const PrefillParams& p, cudaStream_t stream) {
  const int64_t blocks = int64_t(p.N) * p.HV * (128 / (RC_ROWS * RC_WARPS));
  prefill_recurrent_kernel<<<dim3(unsigned(blocks)), RC_WARPS * 32, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace gdnr
