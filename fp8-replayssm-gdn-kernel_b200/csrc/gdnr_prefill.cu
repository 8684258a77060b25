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
//   N (I + A)^T = R,                 A_ij = beta_i rk_i rk_j e^{G_i - G_j} k_i.k_j      (j < i)
//   O = e^G rq S Q^T + N P^T,        P_ij = rq_i rk_j e^{G_i - G_j} q_i.k_j             (j <= i)
//   S = e^{G_C} S + N diag(e^{G_C - G_j} rk_j) K
// (N [V, C] holds the tokens' new values).  All with value rows as the rows of the matrix
// products, so a warp that owns 16 value rows of S keeps S, X, R and N in registers: the
// accumulators of one product are the left operand of the next, and nothing of the chain
// from one state to the next passes through shared memory or waits for another warp.
//
// A CTA has 64 value rows of a head: four consumer warps of 16 rows and four producer warps
// that load the chunk after next and derive A and P of the next one.  N is solved for by
// blocks of 16 tokens: the producers invert I + A's diagonal blocks, the consumers substitute
// (N_b = R_b T_bb^T, then R_i -= N_b A_ib^T for the blocks below).
//
// Rounding: K, Q, V are bf16 as they come.  A float32 matrix meets the tensor cores as a sum
// of narrower ones, so that the float32 state stays within 1e-5 also where keys are alike and
// N is what is left of large terms: S as two bf16 (against K and Q); the weighted N as
// three (its products add up in S, which may be far smaller than their sum of
// sizes); A, T and P, whose entries are at most about one, as two f16, and with them R and N,
// each row brought near one by a power of two first (with two bf16 here the state was
// 1.8e-5 off on such keys).  The output needs it too, although it is bf16: S Q^T and N P^T
// nearly cancel there, and operands rounded once left it 8e-3 off instead of 2e-3.
// Gates are summed in double: differences of float32 prefix sums would cancel under
// strong decay.
constexpr int CK_C = 64;
constexpr int CK_ROWS = 64;
constexpr int CK_THREADS = 256;
constexpr int CK_LDA = 20;  // floats of a row of a diagonal block

struct CkTile {  // one chunk's raw rows, 16-byte chunks swizzled
  uint8_t k[CK_C * 256], q[CK_C * 256], v[CK_C * CK_ROWS * 2];
};
struct CkDerived {
  // diagonal blocks of 16: T = (I + A)^-1 of the block, below them: -A
  uint8_t t_hi[CK_C * 128], t_lo[CK_C * 128], p_hi[CK_C * 128], p_lo[CK_C * 128];
  float beta[CK_C], cx[CK_C], cq[CK_C], cs[CK_C], total;  // beta, beta e^G rk, e^G rq K^-1/2, e^{G_C - G} rk; e^{G_C}
  float pad[15];
};
struct CkSmem {
  CkTile tile[3];
  CkDerived der[2];
  float a[CK_C * CK_LDA];  // A's diagonal blocks: warp w's at rows 16 w
  uint8_t stage[4][CK_C * 48];
  double g[CK_C];
  float g_hi[CK_C], g_lo[CK_C];  // prefix sums of the gates in units of ln 2, in two parts
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
  // tiles of the warp's five units; rows of units 0, 1: block warp, 4: block rb2, 2 and 3: warp 1's own, else rb2
  const int rb2 = warp == 0 ? 3 : (warp == 1 ? 2 : warp);
  const int unit_tile[5] = {2 * warp, 2 * warp + 1, warp < 2 ? 0 : 2 * warp - 3, warp < 2 ? 1 : 2 * warp - 2,
                            warp == 0 ? 2 : (warp == 1 ? 0 : 2 * warp - 1)};
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
      // in two floats: differences of prefix sums are then exact where they matter
      x0 *= 1.4426950408889634, x1 *= 1.4426950408889634;
      const float h0 = float(x0), h1 = float(x1);
      *reinterpret_cast<float2*>(&sm.g_hi[2 * lane]) = make_float2(h0, h1);
      *reinterpret_cast<float2*>(&sm.g_lo[2 * lane]) = make_float2(float(x0 - h0), float(x1 - h1));
    }
    // K K^T and Q K^T on and below the diagonal: 20 tiles of 16 x 8, five a warp, the first two of them the
    // warp's diagonal block; and Q Q^T on the diagonal.  Squared norms are diagonals.
    float kk[5][4], qk[5][4], qq[2][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
#pragma unroll
      for (int j = 0; j < 5; ++j) kk[j][e] = qk[j][e] = 0.f;
      qq[0][e] = qq[1][e] = 0.f;
    }
    const uint32_t ks = smem_addr(tl.k), qs = smem_addr(tl.q);
#pragma unroll
    for (int s = 0; s < 8; s += 2) {
      uint32_t ak1[2][4], aq1[2][4], ak2[2][4], aq2[2][4], bb[5][4], bq[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int ch = (s + i) * 2 + (lane >> 4);
        ldsm_x4(ks + swz<256>(warp * 16 + (lane & 15), ch), ak1[i]);
        ldsm_x4(qs + swz<256>(warp * 16 + (lane & 15), ch), aq1[i]);
        ldsm_x4(ks + swz<256>(rb2 * 16 + (lane & 15), ch), ak2[i]);
        ldsm_x4(qs + swz<256>(rb2 * 16 + (lane & 15), ch), aq2[i]);
        ldsm_x4(qs + swz<256>((2 * warp + i) * 8 + (lane & 7), s * 2 + (lane >> 3)), bq[i]);
      }
#pragma unroll
      for (int u = 0; u < 5; ++u) ldsm_x4(ks + swz<256>(unit_tile[u] * 8 + (lane & 7), s * 2 + (lane >> 3)), bb[u]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t akm[4], aqm[4];  // of units 2 and 3
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          akm[e] = warp == 1 ? ak1[i][e] : ak2[i][e];
          aqm[e] = warp == 1 ? aq1[i][e] : aq2[i][e];
        }
#pragma unroll
        for (int u = 0; u < 5; ++u) {
          mma_bf16(kk[u], u < 2 ? ak1[i] : (u < 4 ? akm : ak2[i]), bb[u][2 * i], bb[u][2 * i + 1]);
          mma_bf16(qk[u], u < 2 ? aq1[i] : (u < 4 ? aqm : aq2[i]), bb[u][2 * i], bb[u][2 * i + 1]);
        }
        mma_bf16(qq[0], aq1[i], bq[0][2 * i], bq[0][2 * i + 1]);
        mma_bf16(qq[1], aq1[i], bq[1][2 * i], bq[1][2 * i + 1]);
      }
    }
    if ((lane >> 3) == (lane & 3)) {  // the thread with elements (g, g) and (g + 8, g + 8) of its diagonal tiles
      const int e = (lane >> 2) & 1, row = warp * 16 + (lane >> 2);
      sm.rk[row] = 1.0f / sqrtf((e ? kk[0][1] : kk[0][0]) + L2_EPS);
      sm.rk[row + 8] = 1.0f / sqrtf((e ? kk[1][3] : kk[1][2]) + L2_EPS);
      sm.rq[row] = 0.08838834764831845f / sqrtf((e ? qq[0][1] : qq[0][0]) + L2_EPS);
      sm.rq[row + 8] = 0.08838834764831845f / sqrtf((e ? qq[1][3] : qq[1][2]) + L2_EPS);
    }
    bar_sync(CK_BAR_PROD, 128);  // prefix sums and norms are in shared memory
    if (tid < CK_C) {
      const float gh = sm.g_hi[tid], gl = sm.g_lo[tid], ch = sm.g_hi[CK_C - 1], cl = sm.g_lo[CK_C - 1];
      const float e = ex2_approx(gh + gl), be = sm.gbeta[tid];
      dv.beta[tid] = be;
      dv.cx[tid] = be * e * sm.rk[tid];
      dv.cq[tid] = e * sm.rq[tid];
      dv.cs[tid] = ex2_approx((ch - gh) + (cl - gl)) * sm.rk[tid];
      if (tid == 0) dv.total = ex2_approx(ch + cl);
    }
#pragma unroll
    for (int u = 0; u < 5; ++u) {
      const int rb = u < 2 ? warp : (u < 4 ? (warp == 1 ? warp : rb2) : rb2);
      const int row0 = rb * 16 + (lane >> 2), col = unit_tile[u] * 8 + 2 * (lane & 3);
      const float2 gh = *reinterpret_cast<const float2*>(&sm.g_hi[col]), gl = *reinterpret_cast<const float2*>(&sm.g_lo[col]),
                   rk = *reinterpret_cast<const float2*>(&sm.rk[col]);
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int row = row0 + 8 * hf;
        const float rh = sm.g_hi[row], rl = sm.g_lo[row], bk = sm.gbeta[row] * sm.rk[row], rq = sm.rq[row];
        const float d0 = ex2_approx((rh - gh.x) + (rl - gl.x)) * rk.x, d1 = ex2_approx((rh - gh.y) + (rl - gl.y)) * rk.y;
        float a0 = bk * d0 * kk[u][2 * hf], a1 = bk * d1 * kk[u][2 * hf + 1];
        float p0 = rq * d0 * qk[u][2 * hf], p1 = rq * d1 * qk[u][2 * hf + 1];
        uint32_t wh, wl;
        const uint32_t at = swz<128>(row, unit_tile[u]) + 4 * (lane & 3);
        if (u < 2) {  // diagonal block: above the diagonal the exponentials may be anything
          p0 = col <= row ? p0 : 0.f;
          p1 = col + 1 <= row ? p1 : 0.f;
          *reinterpret_cast<float2*>(&sm.a[row * CK_LDA + (col & 15)]) = make_float2(col < row ? a0 : 0.f, col + 1 < row ? a1 : 0.f);
        } else {
          split_f16x2(-a0, -a1, wh, wl);
          *reinterpret_cast<uint32_t*>(dv.t_hi + at) = wh;
          *reinterpret_cast<uint32_t*>(dv.t_lo + at) = wl;
        }
        split_f16x2(p0, p1, wh, wl);
        *reinterpret_cast<uint32_t*>(dv.p_hi + at) = wh;
        *reinterpret_cast<uint32_t*>(dv.p_lo + at) = wl;
      }
    }
    __syncwarp();
    {
      // the warp's diagonal block of I + A inverted by substitution, lane = column (both halves of the warp alike)
      const float* ad = sm.a + warp * 16 * CK_LDA;
      const int cl = lane & 15;
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float s0 = i == cl ? 1.f : 0.f, s1 = 0.f;
#pragma unroll
        for (int j = 0; j < i; ++j) {
          if (j & 1)
            s1 -= ad[i * CK_LDA + j] * x[j];
          else
            s0 -= ad[i * CK_LDA + j] * x[j];
        }
        x[i] = s0 + s1;
      }
      // rows of the first half by lanes 0..15, of the second by the others
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float v = lane < 16 ? x[i] : x[8 + i];
        const int row = warp * 16 + i + (lane < 16 ? 0 : 8);
        const __half hi = __float2half_rn(v);
        const uint32_t at = swz<128>(row, warp * 2 + (cl >> 3)) + 2 * (cl & 7);
        *reinterpret_cast<__half*>(dv.t_hi + at) = hi;
        *reinterpret_cast<__half*>(dv.t_lo + at) = __float2half_rn(v - __half2float(hi));
      }
    }
    bar_arrive(CK_BAR_FULL + (c & 1), CK_THREADS);
  }
}

// acc [16, 64] += L M^T for L in two parts as left operands and M [64, 64] lower triangular in two parts
// (rows of 128 bytes): hi hi + lo hi + hi lo (f16).
__device__ __forceinline__ void ck_mul_tri(float (*acc)[4], const uint32_t (*lh)[4], const uint32_t (*ll)[4], uint32_t mh, uint32_t ml,
                                           int lane) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t b[4][4], bl[4][4];
#pragma unroll
    for (int i = j; i < 4; ++i) {
      const uint32_t off = swz<128>(i * 16 + ((lane >> 4) << 3) + (lane & 7), j * 2 + ((lane >> 3) & 1));
      ldsm_x4(mh + off, b[i]);
      ldsm_x4(ml + off, bl[i]);
    }
#pragma unroll
    for (int part = 0; part < 3; ++part)
#pragma unroll
      for (int i = 2 * j; i < 8; ++i) {
        const uint32_t* w = part == 2 ? bl[i >> 1] : b[i >> 1];
        mma_f16(acc[i], part == 1 ? ll[j] : lh[j], w[2 * (i & 1)], w[2 * (i & 1) + 1]);
      }
  }
}

// Two accumulator tiles [16, 8] as a left operand [16, 16], in two parts
__device__ __forceinline__ void ck_left(const float (*x)[4], uint32_t* hi, uint32_t* lo) {
  split_bf16x2(x[0][0], x[0][1], hi[0], lo[0]);
  split_bf16x2(x[0][2], x[0][3], hi[1], lo[1]);
  split_bf16x2(x[1][0], x[1][1], hi[2], lo[2]);
  split_bf16x2(x[1][2], x[1][3], hi[3], lo[3]);
}

__device__ __forceinline__ void ck_left_f16(const float (*x)[4], uint32_t* hi, uint32_t* lo) {
  split_f16x2(x[0][0], x[0][1], hi[0], lo[0]);
  split_f16x2(x[0][2], x[0][3], hi[1], lo[1]);
  split_f16x2(x[1][0], x[1][1], hi[2], lo[2]);
  split_f16x2(x[1][2], x[1][3], hi[3], lo[3]);
}

// A power of two that brings a row's largest value (over the four lanes that hold the row) into
// [2^4, 2^5), and its inverse
__device__ __forceinline__ void ck_row_scale(float top, float& up, float& down) {
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  const int e = min(max(int(__float_as_uint(top) >> 23), 8), 250);
  up = __uint_as_float(uint32_t(258 - e) << 23);
  down = __uint_as_float(uint32_t(e - 4) << 23);
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
      ck_left(S + 2 * s, hi, lo);
      // products that add to the same tile are kept eight apart: one takes about four times as long as it keeps the unit
#pragma unroll
      for (int jj = 0; jj < 4; jj += 2) {
        uint32_t bk[2][4], bq[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t off = swz<256>((jj + j) * 16 + ((lane >> 4) << 3) + (lane & 7), s * 2 + ((lane >> 3) & 1));
          ldsm_x4(ks + off, bk[j]);
          ldsm_x4(qs + off, bq[j]);
        }
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            mma_bf16(X[2 * jj + j], part ? lo : hi, bk[j >> 1][2 * (j & 1)], bk[j >> 1][2 * (j & 1) + 1]);
            mma_bf16(O[2 * jj + j], part ? lo : hi, bq[j >> 1][2 * (j & 1)], bq[j >> 1][2 * (j & 1) + 1]);
          }
      }
    }
    // R = beta V^T - (beta e^G rk) X
    float top0 = 0.f, top1 = 0.f;
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
        x[0] = be.x * v0f.x - cx.x * x[0], x[1] = be.y * v0f.y - cx.y * x[1];
        x[2] = be.x * v1f.x - cx.x * x[2], x[3] = be.y * v1f.y - cx.y * x[3];
        top0 = fmaxf(top0, fmaxf(fabsf(x[0]), fabsf(x[1])));
        top1 = fmaxf(top1, fmaxf(fabsf(x[2]), fabsf(x[3])));
        o[0] *= cq.x, o[1] *= cq.y, o[2] *= cq.x, o[3] *= cq.y;
      }
    }
    // rows to at most 2^5 (N stays far below 2^15 then: keys are of unit length and beta at most one)
    float up0, down0, up1, down1;
    ck_row_scale(top0, up0, down0);
    ck_row_scale(top1, up1, down1);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      X[j][0] *= up0, X[j][1] *= up0, X[j][2] *= up1, X[j][3] *= up1;
      O[j][0] *= up0, O[j][1] *= up0, O[j][2] *= up1, O[j][3] *= up1;
    }
    float N[8][4];
    uint32_t nh[4][4], nl[4][4];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) N[j][e] = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // column j of blocks: T_jj, then -A_ij below it
      uint32_t b[4][4], bl[4][4], rh[4], rl[4];
#pragma unroll
      for (int i = j; i < 4; ++i) {
        const uint32_t off = swz<128>(i * 16 + ((lane >> 4) << 3) + (lane & 7), j * 2 + ((lane >> 3) & 1));
        ldsm_x4(th + off, b[i]);
        ldsm_x4(tlo + off, bl[i]);
      }
      ck_left_f16(X + 2 * j, rh, rl);
#pragma unroll
      for (int part = 0; part < 3; ++part)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          mma_f16(N[2 * j + i], part == 1 ? rl : rh, (part == 2 ? bl : b)[j][2 * i], (part == 2 ? bl : b)[j][2 * i + 1]);
      ck_left_f16(N + 2 * j, nh[j], nl[j]);
#pragma unroll
      for (int part = 0; part < 3; ++part)
#pragma unroll
        for (int i = 2 * j + 2; i < 8; ++i) {
          const uint32_t* w = (part == 2 ? bl : b)[i >> 1];
          mma_f16(X[i], part == 1 ? nl[j] : nh[j], w[2 * (i & 1)], w[2 * (i & 1) + 1]);
        }
    }
    // the state first: the next chunk waits for it
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
        split3_bf16x2(x[0] * (cs.x * down0), x[1] * (cs.y * down0), hi[2 * hf], lo[2 * hf], rest[2 * hf]);
        split3_bf16x2(x[2] * (cs.x * down1), x[3] * (cs.y * down1), hi[2 * hf + 1], lo[2 * hf + 1], rest[2 * hf + 1]);
      }
#pragma unroll
      for (int nn = 0; nn < 8; nn += 4) {
        uint32_t b[4][4];
#pragma unroll
        for (int n = 0; n < 4; ++n) ldsm_x4_t(ks + swz<256>(j * 16 + (lane & 15), (nn + n) * 2 + (lane >> 4)), b[n]);
#pragma unroll
        for (int part = 0; part < 3; ++part)
#pragma unroll
          for (int n = 0; n < 8; ++n)
            mma_bf16(S[2 * nn + n], part == 0 ? hi : (part == 1 ? lo : rest), b[n >> 1][2 * (n & 1)], b[n >> 1][2 * (n & 1) + 1]);
      }
    }
    ck_mul_tri(O, nh, nl, ph, pl, lane);
    if (c + 2 < chunks) bar_arrive(CK_BAR_EMPTY + (c & 1), CK_THREADS);
    // O^T to token rows through the warp's own staging rows (48 bytes apart: no bank twice)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      stsm_x4_t(stage + (j * 16 + ((lane >> 4) << 3) + (lane & 7)) * 48 + ((lane >> 3) & 1) * 16, cvt_bf16x2(O[2 * j][0] * down0, O[2 * j][1] * down0),
                cvt_bf16x2(O[2 * j][2] * down1, O[2 * j][3] * down1), cvt_bf16x2(O[2 * j + 1][0] * down0, O[2 * j + 1][1] * down0),
                cvt_bf16x2(O[2 * j + 1][2] * down1, O[2 * j + 1][3] * down1));
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
