// The gated delta rule over ragged sequences (gdnr_gdn_prefill).
//
//   S_t = e^{g_t} S_{t-1} + d_t k_t^T,   d_t = beta_t (v_t - e^{g_t} S_{t-1} k_t),   o_t = S_t q_t
//
// per value head, S [V, K] float32, with k = k_raw / sqrt(|k_raw|^2 + eps), q likewise times
// K^-1/2, g = -exp(A_log) softplus(a + dt_bias), beta = sigmoid(b).
#include "gdnr_device.cuh"
#include "gdnr_hybrid.h"

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

}  // namespace

cudaError_t launch_prefill_recurrent(const PrefillParams& p, cudaStream_t stream) {
  const int64_t blocks = int64_t(p.N) * p.HV * (128 / (RC_ROWS * RC_WARPS));
  prefill_recurrent_kernel<<<dim3(unsigned(blocks)), RC_WARPS * 32, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace gdnr
