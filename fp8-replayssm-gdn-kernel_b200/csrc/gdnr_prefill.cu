// The gated delta rule over ragged sequences (gdnr_gdn_prefill).
//
//   S_t = e^{g_t} S_{t-1} + d_t k_t^T,   d_t = beta_t (v_t - e^{g_t} S_{t-1} k_t),   o_t = S_t q_t
//
// per value head, S [V, K] float32, with k = k_raw / sqrt(|k_raw|^2 + eps), q likewise times
// K^-1/2, g = -exp(A_log) softplus(a + dt_bias), beta = sigmoid(b).
#include "gdnr_device.cuh"
#include "gdnr_hybrid.h"
#include "gdnr_tc.cuh"

#include <algorithm>

namespace gdnr {

namespace {

// log(1 + e^x), x itself above the threshold the gates of the decode step use.
__device__ __forceinline__ float softplus_gate(float x) { return x > SOFTPLUS_THRESHOLD ? x : log1pf(expf(x)); }

__device__ __forceinline__ float sigmoid_f(float x) { return 1.0f / (1.0f + expf(-x)); }

// load_scalar in two steps, so that a thread's loads can be on their way together
__device__ __forceinline__ uint32_t load_word(const void* p, int64_t i, int dtype) {
  return dtype == GDNR_F32 ? static_cast<const uint32_t*>(p)[i] : static_cast<const uint16_t*>(p)[i];
}

__device__ __forceinline__ float word_value(uint32_t w, int dtype) {
  return dtype == GDNR_F32 ? __uint_as_float(w) : (dtype == GDNR_BF16 ? bf16_to_f(uint16_t(w)) : __half2float(__ushort_as_half(uint16_t(w))));
}

// ---------------------------------------------------------------- recurrent form
// One warp owns 8 value rows of S in registers (lane: 4 key columns of each), a CTA 32
// rows, so a head is four CTAs and a batch of single tokens reads and writes each state
// once, in 512-byte row pieces.  What does not depend on the state (inverse norms, q.k, gates) is
// made for up to 16 tokens at a time, the tokens shared by the warps, so that a token
// costs its own chain only: S k and S q, both from the state before the update
// (o = e^g S q + d (k.q)), one chain of shuffles, the update.  The sums of 8 rows over 32 lanes are
// folded together: 4 + 2 + 1 exchanges halve the rows a lane holds, 2 more finish the
// sum, 9 shuffles instead of 40.
// 64 single tokens of 32 heads: 43 us, 6.3 TB/s of the 270 MB of states read and written; 24 sequences of 2 to 7
// tokens: 32 us a call (45 us with the factors made token by token in the chain).
constexpr int RC_ROWS = 8;
constexpr int RC_WARPS = 4;
constexpr int RC_BLOCK = 16;

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

struct RcSmem {
  uint2 q[RC_BLOCK][32], k[RC_BLOCK][32];  // raw rows, a lane's four elements
  uint16_t v[RC_BLOCK][RC_ROWS * RC_WARPS];
  float alpha[RC_BLOCK], beta[RC_BLOCK], rk[RC_BLOCK], rq[RC_BLOCK], qk[RC_BLOCK];
};

__global__ void __launch_bounds__(RC_WARPS * 32) prefill_recurrent_kernel(const __grid_constant__ PrefillParams p) {
  __shared__ RcSmem sm;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int PARTS = 128 / (RC_ROWS * RC_WARPS);
  const int part = blockIdx.x % PARTS, nh = blockIdx.x / PARTS;
  const int n = nh / p.HV, hv = nh - n * p.HV, h = hv / (p.HV / p.H);
  const int part0 = part * (RC_ROWS * RC_WARPS), row0 = part0 + warp * RC_ROWS;
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
  for (int t0 = r.begin; t0 < r.end; t0 += RC_BLOCK) {
    const int count = min(RC_BLOCK, r.end - t0);
    if (t0 > r.begin) __syncthreads();  // the block before has been used
    if (tid >= 64 && tid < 64 + count) {  // gates: a thread a token
      const int i = tid - 64, t = t0 + i;
      const float a = load_scalar(p.a, int64_t(t) * p.a_st + int64_t(hv) * p.a_sh, p.a_dt) + p.dt_bias[hv * p.db_s];
      const float b = load_scalar(p.b, int64_t(t) * p.b_st + int64_t(hv) * p.b_sh, p.b_dt);
      sm.alpha[i] = expf(-expf(p.a_log[hv * p.al_s]) * softplus_gate(a));
      sm.beta[i] = sigmoid_f(b);
    }
    for (int i = warp; i < count; i += RC_WARPS) {
      const uint16_t* m = p.mixed + int64_t(t0 + i) * p.mx_s;
      const uint2 q = *reinterpret_cast<const uint2*>(m + h * 128 + lane * 4), k = *reinterpret_cast<const uint2*>(m + (p.H + h) * 128 + lane * 4);
      sm.v[i][lane] = m[(2 * p.H + hv) * 128 + part0 + lane];
      sm.q[i][lane] = q;
      sm.k[i][lane] = k;
      const float2 q01 = bf16x2_to_f2(q.x), q23 = bf16x2_to_f2(q.y), k01 = bf16x2_to_f2(k.x), k23 = bf16x2_to_f2(k.y);
      float qq = q01.x * q01.x + q01.y * q01.y + q23.x * q23.x + q23.y * q23.y;
      float kk = k01.x * k01.x + k01.y * k01.y + k23.x * k23.x + k23.y * k23.y;
      float qk = q01.x * k01.x + q01.y * k01.y + q23.x * k23.x + q23.y * k23.y;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        qq += __shfl_xor_sync(0xffffffffu, qq, o);
        kk += __shfl_xor_sync(0xffffffffu, kk, o);
        qk += __shfl_xor_sync(0xffffffffu, qk, o);
      }
      if (lane == 0) {
        const float rk = rsqrtf(kk + L2_EPS), rq = 0.08838834764831845f * rsqrtf(qq + L2_EPS);
        sm.rk[i] = rk, sm.rq[i] = rq, sm.qk[i] = qk * rk * rq;
      }
    }
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < count; ++i) {
      const uint2 q = sm.q[i][lane], k = sm.k[i][lane];
      const float2 q01 = bf16x2_to_f2(q.x), q23 = bf16x2_to_f2(q.y), k01 = bf16x2_to_f2(k.x), k23 = bf16x2_to_f2(k.y);
      float sk[RC_ROWS], sq[RC_ROWS];
#pragma unroll
      for (int j = 0; j < RC_ROWS; ++j) {
        sk[j] = S[j].x * k01.x + S[j].y * k01.y + S[j].z * k23.x + S[j].w * k23.y;
        sq[j] = S[j].x * q01.x + S[j].y * q01.y + S[j].z * q23.x + S[j].w * q23.y;
      }
      const float alpha = sm.alpha[i], rk = sm.rk[i];
      const float my_sk = fold8(sk, lane), my_sq = fold8(sq, lane);
      const float d = sm.beta[i] * (bf16_to_f(sm.v[i][warp * RC_ROWS + (lane >> 2)]) - alpha * rk * my_sk);
      if ((lane & 3) == 0)
        p.out[int64_t(t0 + i) * p.o_st + int64_t(hv) * p.o_sh + my_row] = f_to_bf16(alpha * sm.rq[i] * my_sq + d * sm.qk[i]);
      const float dk = d * rk;
#pragma unroll
      for (int j = 0; j < RC_ROWS; ++j) {
        const float dj = __shfl_sync(0xffffffffu, dk, j * 4);
        S[j].x = alpha * S[j].x + dj * k01.x;
        S[j].y = alpha * S[j].y + dj * k01.y;
        S[j].z = alpha * S[j].z + dj * k23.x;
        S[j].w = alpha * S[j].w + dj * k23.y;
      }
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
// (N [V, C] holds the tokens' new values).
//
// Two kernels.  The first makes what does not depend on the state, for all chunks at once: T = (I + A)^-1
// or A with its diagonal blocks of 16 tokens inverted, P, and the factors of each token, an image of
// 21 KB a chunk and head in the layout the second one's shared memory has.  The second
// walks the chunks of a sequence, with value rows as the rows of the matrix products, in one of two forms:
//   tcgen05: a head's 128 value rows are the lanes of tensor memory, where S stays; N = R T^T.
//   warp-level, where few heads leave multiprocessors over: a head on four of them.  Two warps share 16 value rows
//   and keep S, X, R and N in registers; the accumulators of one product are the left operand of the
//   next.  N is solved for by blocks (N_b = R_b T_bb^T, then R_i -= N_b A_ib^T for the blocks below): the whole
//   T gained nothing here (0.353 ms a 8192-token prompt, not 0.361, for 8 us more in the first kernel).
//
// Rounding: K, Q, V are bf16 as they come.  A float32 matrix meets the tensor cores as a sum
// of narrower ones, so that the float32 state stays within 1e-5 also where keys are alike and
// N is what is left of large terms: S as two bf16 (against K and Q); the weighted N as
// three (its products add up in S, which may be far smaller than their sum of
// sizes); A, T and P, whose entries are at most one, as two f16 of 2^14 times them, and with them R and N,
// each row of R brought to 2^8 by a power of two first (with two bf16 here the state was
// 1.8e-5 off on such keys).  f16 ends at 2^-24: an entry of T is exact to 2^-39, one of R to 2^-34 of its row's largest
// in the chunk (2^-25 and 2^-30 without the powers: a state that little was written to, behind large and decayed
// values, had errors of 1e-4).  The output needs it too, although it is bf16: S Q^T and N P^T
// nearly cancel there, and operands rounded once left it 8e-3 off instead of 2e-3.
// Gates are summed in double: differences of float32 prefix sums would cancel under
// strong decay.
constexpr int CK_C = 64;

// Lower triangular [C, C] of f16 as its ten blocks of 16 x 16, column by column: rows of 32 bytes whose two
// 16-byte halves change places every four rows (the 32-byte swizzle: eight rows' equal halves cover all banks, and
// a column's blocks are one right operand of the tensor cores).
constexpr int CK_TRI = 10 * 512;
__host__ __device__ constexpr int ck_block(int i, int j) { return (4 * j - j * (j - 1) / 2 + i - j) * 512; }
__device__ __forceinline__ uint32_t ck_in_block(int row, int half) { return row * 32 + ((half ^ ((row >> 2) & 1)) << 4); }

constexpr float CK_UP = 16384.f, CK_DOWN = 1.f / CK_UP;

struct CkImage {
  // t: diagonal blocks: (I + A)^-1 of the block, below them: -A; or (whole) T = (I + A)^-1; t and p times CK_UP
  uint8_t t_hi[CK_TRI], t_lo[CK_TRI], p_hi[CK_TRI], p_lo[CK_TRI];
  float beta[CK_C], cx[CK_C], cq[CK_C], cs[CK_C], total;  // beta, -beta e^G rk, e^G rq K^-1/2, e^{G_C - G} rk; e^{G_C}
  uint32_t made;  // 1: all of it is there; 0: the first kernel's wait gave up
  float pad[14];
};
static_assert(sizeof(CkImage) == CK_IMAGE_BYTES && sizeof(CkImage) % 16 == 0, "copied in bulk");

// 64 rows of 128 bf16 as two TMA boxes of 64 columns, 128-byte swizzle: 16-byte chunk c of row r
__device__ __forceinline__ uint32_t ck_at(int row, int c) { return uint32_t(c >> 3) * 8192u + swz<128>(row, c & 7); }

__device__ __forceinline__ void ck_tma(uint32_t dst, const CUtensorMap* map, int col, int row, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(col), "r"(row), "r"(smem_addr(bar))
      : "memory");
}

// The chunks of sequence n have the numbers ck_first(n) ..; they do not overlap, and end below T / C + N.
__device__ __forceinline__ int ck_first(int begin, int n) { return begin / CK_C + n; }

// Rows from `valid` on of a tile: what lies past the sequence's end belongs to others (it may be NaN)
__device__ __forceinline__ void ck_zero_rows(uint8_t* tile, int boxes, int valid, int tid, int threads) {
  for (int i = tid; i < boxes * (CK_C - valid) * 8; i += threads) {
    const int box = i / ((CK_C - valid) * 8), j = i % ((CK_C - valid) * 8);
    *reinterpret_cast<uint4*>(tile + box * 8192 + (valid + j / 8) * 128 + (j & 7) * 16) = make_uint4(0, 0, 0, 0);
  }
}

// Two accumulator tiles [16, 8] as a left operand [16, 16], in two parts
__device__ __forceinline__ void ck_left_f16(const float (*x)[4], uint32_t* hi, uint32_t* lo) {
  split_f16x2(x[0][0], x[0][1], hi[0], lo[0]);
  split_f16x2(x[0][2], x[0][3], hi[1], lo[1]);
  split_f16x2(x[1][0], x[1][1], hi[2], lo[2]);
  split_f16x2(x[1][2], x[1][3], hi[3], lo[3]);
}

// Two neighbouring floats of a factor
__device__ __forceinline__ uint64_t pair_at(const float* p) { return *reinterpret_cast<const uint64_t*>(p); }

// ---------------------------------------------------------------- chunked form, first kernel
constexpr int CD_THREADS = 256;
constexpr int CD_LDA = 20;  // floats of a row of a diagonal block

struct CdSmem {
  union {
    struct {
      uint8_t k[CK_C * 256], q[CK_C * 256];
    };
    CkImage img[2];  // once the products are in registers
  };
  float a[2][CK_C * CD_LDA];  // -A's diagonal blocks of two heads: warp w's at rows 16 w
  float g_hi[2][CK_C], g_lo[2][CK_C], gbeta[2][CK_C];  // prefix sums of the gates in units of ln 2, in two parts
  float rk[CK_C], rq[CK_C];
  uint64_t bar;
};

// One CTA a chunk and key head; its value heads share the products of the raw rows.  Bound by
// instructions and barriers (three CTAs a multiprocessor; a 8192-token prompt of 16 / 32 heads: 50 us, 88 MB of
// images; with the gates' loads one after another 56 us).  The first four warps make A (rows of K against K) and invert its diagonal blocks, the others make P
// (rows of Q against K) and the factors.
__global__ void __launch_bounds__(CD_THREADS, 3) prefill_derive_kernel(const __grid_constant__ PrefillParams p,
                                                                       const __grid_constant__ CUtensorMap map) {
  extern __shared__ uint8_t raw[];
  CdSmem& sm = *reinterpret_cast<CdSmem*>(raw + (-smem_addr(raw) & 1023u));
  const int tid = threadIdx.x, lane = tid & 31, warp = (tid >> 5) & 3;
  griddep_launch();  // the second kernel's CTAs may be set up once every one of these has begun
  const int id = blockIdx.x / p.H, h = blockIdx.x - id * p.H, group = p.HV / p.H;
  // the last sequence whose first chunk is not after this one
  int lo = 0, hi = p.N - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (ck_first(min(max(p.cu[mid], 0), p.T), mid) <= id)
      lo = mid;
    else
      hi = mid - 1;
  }
  const int n = lo;
  const SeqRange r = prefill_seq(p, n);
  const int c = id - ck_first(r.begin, n);
  if (r.slot < 0 || c < 0 || r.begin + c * CK_C >= r.end) return;
  const int t0 = r.begin + c * CK_C, valid = min(CK_C, r.end - t0);

  if (tid == 0) {
    mbar_init(&sm.bar, 1);
    fence_mbar_init();
    mbar_arrive_expect_tx(&sm.bar, 2 * CK_C * 256);
    for (int b = 0; b < 2; ++b) {
      ck_tma(smem_addr(sm.q) + b * 8192, &map, h * 128 + b * 64, t0, &sm.bar);
      ck_tma(smem_addr(sm.k) + b * 8192, &map, (p.H + h) * 128 + b * 64, t0, &sm.bar);
    }
  }
  const bool of_q = tid >= 128;
  // gates of up to two value heads, one warp each, lane: two tokens; tokens past the end neither decay nor write
  auto make_gates = [&](int e0) {
    const int e = tid >> 5;
    if (e >= 2 || e0 + e >= group) return;
    const int hv = h * group + e0 + e;
    const float a_log = p.a_log[hv * p.al_s], dtb = p.dt_bias[hv * p.db_s];
    uint32_t aw[2], bw[2];  // all loads before their first use: one after another the CTA took 10.4 us instead of 8
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t t = t0 + min(2 * lane + i, valid - 1);
      aw[i] = load_word(p.a, t * p.a_st + int64_t(hv) * p.a_sh, p.a_dt);
      bw[i] = load_word(p.b, t * p.b_st + int64_t(hv) * p.b_sh, p.b_dt);
    }
    const float neg_a = -expf(a_log);
    double x[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = 2 * lane + i;
      float g = 0.f, be = 0.f;
      if (t < valid) {
        g = neg_a * softplus_gate(word_value(aw[i], p.a_dt) + dtb);
        g = g < -1e4f ? -1e4f : g;  // e^g is 0 below; a sum with an infinity would have no differences
        be = sigmoid_f(word_value(bw[i], p.b_dt));
      }
      x[i] = double(g);
      sm.gbeta[e][t] = be;
    }
    x[1] += x[0];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, x[1], o);
      if (lane >= o) x[0] += y, x[1] += y;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      // in two floats: differences of prefix sums are then exact where they matter
      const double y = x[i] * 1.4426950408889634;
      const float hi = float(y);
      sm.g_hi[e][2 * lane + i] = hi;
      sm.g_lo[e][2 * lane + i] = float(y - hi);
    }
  };
  // What lies below the diagonal blocks T_ii of T = (I + A)^-1, in the image, by halves of 32, then of 64 tokens: the
  // block below two inverses is T_low (-A) T_top.  Two warps a head.  (12 ragged prompts of 32 heads: the kernel takes
  // 41 us without it, 49 us with it, and 58 us with the products in float32 on the other units.)
  auto invert_below = [&](int e0) {
    const int e = warp >> 1, w = warp & 1;
    const bool mine = e0 + e < group;
    CkImage& img = sm.img[e];
    const uint32_t hi = smem_addr(img.t_hi), lo = smem_addr(img.t_lo), in = ck_in_block(lane & 15, lane >> 4);
    // acc += L R, R block (i, j) of the image
    auto times = [&](float* acc, const uint32_t* lh, const uint32_t* ll, int i, int j) {
      uint32_t rh[4], rl[4];
      ldsm_x4_t(hi + ck_block(i, j) + in, rh);
      ldsm_x4_t(lo + ck_block(i, j) + in, rl);
#pragma unroll
      for (int q = 0; q < 3; ++q)
#pragma unroll
        for (int t = 0; t < 2; ++t) mma_f16(acc + 4 * t, q == 1 ? ll : lh, (q == 2 ? rl : rh)[2 * t], (q == 2 ? rl : rh)[2 * t + 1]);
    };
    auto times_block = [&](float* acc, int li, int lj, int i, int j) {
      uint32_t lh[4], ll[4];
      ldsm_x4(hi + ck_block(li, lj) + in, lh);
      ldsm_x4(lo + ck_block(li, lj) + in, ll);
      times(acc, lh, ll, i, j);
    };
    auto emit = [&](const float* acc, int i, int j) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {  // tile k / 2, rows + 8 (k % 2)
        uint32_t wh, wl;
        split_f16x2(acc[2 * k], acc[2 * k + 1], wh, wl);
        const uint32_t at = ck_block(i, j) + ck_in_block(lane >> 2, k >> 1) + 4 * (lane & 3) + (k & 1) * 256;
        *reinterpret_cast<uint32_t*>(img.t_hi + at) = wh;
        *reinterpret_cast<uint32_t*>(img.t_lo + at) = wl;
      }
    };
    // T_low (-A) comes as CK_UP^2 times it; 2^10 times it as a left operand (its entries: at most 33, sums of T's)
    auto scale = [&](float* v, float f) {
#pragma unroll
      for (int k = 0; k < 8; k += 2) scale2(v + k, pack2(f, f));
    };
    constexpr float LEFT = 1024.f, TO_LEFT = LEFT / (CK_UP * CK_UP), FROM_LEFT = 1.f / LEFT;
    float x[2][8] = {}, y[2][8] = {};
    uint32_t wh[4], wl[4];
    bar_sync(1, 128);
    if (mine) {
      times_block(x[0], 2 * w + 1, 2 * w + 1, 2 * w + 1, 2 * w);  // T_low (-A)
      scale(x[0], TO_LEFT);
      ck_left_f16(reinterpret_cast<const float(*)[4]>(x[0]), wh, wl);
      times(y[0], wh, wl, 2 * w, 2 * w);
      scale(y[0], FROM_LEFT);
      __syncwarp();
      emit(y[0], 2 * w + 1, 2 * w);
    }
    bar_sync(1, 128);
    // row 2 + w
#pragma unroll
    for (int k = 0; k < 8; ++k) x[0][k] = x[1][k] = y[0][k] = 0.f;
    if (mine) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        times_block(x[j], 2 + w, 2, 2, j);
        if (w) times_block(x[j], 3, 3, 3, j);
        scale(x[j], TO_LEFT);
        ck_left_f16(reinterpret_cast<const float(*)[4]>(x[j]), wh, wl);
        times(y[0], wh, wl, j, 0);
        if (j) times(y[1], wh, wl, 1, 1);
      }
    }
    bar_sync(1, 128);
    if (mine) {
      scale(y[0], FROM_LEFT);
      scale(y[1], FROM_LEFT);
      emit(y[0], 2 + w, 0);
      emit(y[1], 2 + w, 1);
    }
  };
  make_gates(0);  // while the rows are on their way
  __syncthreads();  // the barrier is initialised
  const bool ok = mbar_wait_bounded(&sm.bar, 0, p.err);
  if (__syncthreads_or(!ok)) {
    // the second kernel must not take what lies in the workspace for this chunk's images
    for (int e = tid; e < group; e += CD_THREADS)
      reinterpret_cast<CkImage*>(p.images + (int64_t(id) * p.HV + h * group + e) * CK_IMAGE_BYTES)->made = 0;
    if (tid == 0) drain(&sm.bar, 1, 1);
    return;
  }
  if (valid < CK_C) {
    ck_zero_rows(sm.k, 2, valid, tid, CD_THREADS);
    ck_zero_rows(sm.q, 2, valid, tid, CD_THREADS);
    __syncthreads();
  }
  // K K^T or Q K^T on and below the diagonal: 20 tiles of 16 x 8, five a warp, the first two of them the warp's
  // diagonal block; rows of units 0, 1: block warp, 4: block rb2, 2 and 3: warp 1's own, else rb2.  And Q Q^T on
  // the diagonal.  Squared norms are diagonals.
  const int rb2 = warp == 0 ? 3 : (warp == 1 ? 2 : warp);
  const int unit_tile[5] = {2 * warp, 2 * warp + 1, warp < 2 ? 0 : 2 * warp - 3, warp < 2 ? 1 : 2 * warp - 2,
                            warp == 0 ? 2 : (warp == 1 ? 0 : 2 * warp - 1)};
  float m[5][4], qq[2][4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
#pragma unroll
    for (int j = 0; j < 5; ++j) m[j][e] = 0.f;
    qq[0][e] = qq[1][e] = 0.f;
  }
  const uint32_t ks = smem_addr(sm.k), qs = smem_addr(sm.q), as = of_q ? qs : ks;
#pragma unroll
  for (int s = 0; s < 8; s += 2) {
    uint32_t a1[2][4], a2[2][4], bb[5][4], bq[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int ch = (s + i) * 2 + (lane >> 4);
      ldsm_x4(as + ck_at(warp * 16 + (lane & 15), ch), a1[i]);
      ldsm_x4(as + ck_at(rb2 * 16 + (lane & 15), ch), a2[i]);
    }
#pragma unroll
    for (int u = 0; u < 5; ++u) ldsm_x4(ks + ck_at(unit_tile[u] * 8 + (lane & 7), s * 2 + (lane >> 3)), bb[u]);
    if (of_q) {
#pragma unroll
      for (int i = 0; i < 2; ++i) ldsm_x4(qs + ck_at((2 * warp + i) * 8 + (lane & 7), s * 2 + (lane >> 3)), bq[i]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mma_bf16(qq[0], a1[i], bq[0][2 * i], bq[0][2 * i + 1]);
        mma_bf16(qq[1], a1[i], bq[1][2 * i], bq[1][2 * i + 1]);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t am[4];  // of units 2 and 3
#pragma unroll
      for (int e = 0; e < 4; ++e) am[e] = warp == 1 ? a1[i][e] : a2[i][e];
#pragma unroll
      for (int u = 0; u < 5; ++u) mma_bf16(m[u], u < 2 ? a1[i] : (u < 4 ? am : a2[i]), bb[u][2 * i], bb[u][2 * i + 1]);
    }
  }
  if ((lane >> 3) == (lane & 3)) {  // the thread with elements (g, g) and (g + 8, g + 8) of its diagonal tiles
    const int e = (lane >> 2) & 1, row = warp * 16 + (lane >> 2);
    const float x0 = of_q ? (e ? qq[0][1] : qq[0][0]) : (e ? m[0][1] : m[0][0]);
    const float x1 = of_q ? (e ? qq[1][3] : qq[1][2]) : (e ? m[1][3] : m[1][2]);
    const float gain = of_q ? 0.08838834764831845f : 1.0f;
    (of_q ? sm.rq : sm.rk)[row] = gain * rsqrtf(x0 + L2_EPS);
    (of_q ? sm.rq : sm.rk)[row + 8] = gain * rsqrtf(x1 + L2_EPS);
  }
  __syncthreads();  // gates and norms
  // what all heads share: the products times both norms (and the sign of -A)
  const int rbm = warp == 1 ? warp : rb2;
  const float gain = of_q ? CK_UP : -CK_UP;
  const float* rn = of_q ? sm.rq : sm.rk;
#pragma unroll
  for (int u = 0; u < 5; ++u) {
    const int row = (u < 2 ? warp : (u < 4 ? rbm : rb2)) * 16 + (lane >> 2);
    const uint64_t rk = pair_at(&sm.rk[unit_tile[u] * 8 + 2 * (lane & 3)]);
    const float f0 = gain * rn[row], f1 = gain * rn[row + 8];
    scale2(m[u], mul2(rk, pack2(f0, f0)));
    scale2(m[u] + 2, mul2(rk, pack2(f1, f1)));
  }
  for (int e0 = 0; e0 < group; e0 += 2) {
    if (e0) {  // the two images have left
      if (tid == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      make_gates(e0);
      __syncthreads();
    }
    for (int e = 0; e < 2 && e0 + e < group; ++e) {
      CkImage& img = sm.img[e];
      const float *g_hi = sm.g_hi[e], *g_lo = sm.g_lo[e], *gbeta = sm.gbeta[e];
      if (of_q && tid < 128 + CK_C) {
        const int gt = tid - 128;
        const float gh = g_hi[gt], gl = g_lo[gt], ch = g_hi[CK_C - 1], cl = g_lo[CK_C - 1];
        const float ex = ex2_approx(gh + gl), be = gbeta[gt];
        img.beta[gt] = be;
        img.cx[gt] = -be * ex * sm.rk[gt];
        img.cq[gt] = ex * sm.rq[gt];
        img.cs[gt] = ex2_approx((ch - gh) + (cl - gl)) * sm.rk[gt];
        if (gt == 0) img.total = ex2_approx(ch + cl), img.made = 1;
      }
      // the rows of the three blocks that this thread's units lie in
      float rh[3][2], rl[3][2], rb[3][2];
#pragma unroll
      for (int k = 0; k < 3; ++k)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int row = (k == 0 ? warp : (k == 1 ? rbm : rb2)) * 16 + (lane >> 2) + 8 * hf;
          rh[k][hf] = g_hi[row], rl[k][hf] = g_lo[row], rb[k][hf] = of_q ? 1.f : gbeta[row];
        }
      const uint64_t minus = pack2(-1.f, -1.f);
#pragma unroll
      for (int u = 0; u < 5; ++u) {
        const int k = u < 2 ? 0 : (u < 4 ? 1 : 2), block_row = k == 0 ? warp : (k == 1 ? rbm : rb2);
        const int col = unit_tile[u] * 8 + 2 * (lane & 3);
        const uint64_t gh = pair_at(&g_hi[col]), gl = pair_at(&g_lo[col]);
        // (rows r and r + 8 have their halves in the same order)
        const uint32_t at = ck_block(block_row, unit_tile[u] >> 1) + ck_in_block(lane >> 2, unit_tile[u] & 1) + 4 * (lane & 3);
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const float2 d = unpack2(add2(fma2(gh, minus, pack2(rh[k][hf], rh[k][hf])), fma2(gl, minus, pack2(rl[k][hf], rl[k][hf]))));
          const uint64_t f = of_q ? pack2(m[u][2 * hf], m[u][2 * hf + 1]) : mul2(pack2(m[u][2 * hf], m[u][2 * hf + 1]), pack2(rb[k][hf], rb[k][hf]));
          float2 x = unpack2(mul2(pack2(ex2_approx(d.x), ex2_approx(d.y)), f));
          if (u < 2) {  // diagonal block: above the diagonal the exponentials may be anything
            const int row = (lane >> 2) + 8 * hf, c = (unit_tile[u] & 1) * 8 + 2 * (lane & 3), last = of_q ? row : row - 1;
            x.x = c <= last ? x.x : 0.f;
            x.y = c < last ? x.y : 0.f;
            if (!of_q) *reinterpret_cast<float2*>(&sm.a[e][(warp * 16 + row) * CD_LDA + c]) = make_float2(x.x * CK_DOWN, x.y * CK_DOWN);
          }
          if (u >= 2 || of_q) {
            uint32_t wh, wl;
            split_f16x2(x.x, x.y, wh, wl);
            *reinterpret_cast<uint32_t*>((of_q ? img.p_hi : img.t_hi) + at + hf * 256) = wh;
            *reinterpret_cast<uint32_t*>((of_q ? img.p_lo : img.t_lo) + at + hf * 256) = wl;
          }
        }
      }
    }
    if (!of_q) {
      __syncwarp();
      // the warp's diagonal blocks of I + A (sm.a holds -A) inverted by substitution: half a warp a head, lane = column
      const int e = lane >> 4, cl = lane & 15;
      const float* ad = sm.a[e] + warp * 16 * CD_LDA;
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float s[4] = {i == cl ? CK_UP : 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < i; j += 4) {
          const float4 v = *reinterpret_cast<const float4*>(&ad[i * CD_LDA + j]);
          s[0] += v.x * x[j];
          if (j + 1 < i) s[1] += v.y * x[j + 1];
          if (j + 2 < i) s[2] += v.z * x[j + 2];
          if (j + 3 < i) s[3] += v.w * x[j + 3];
        }
        x[i] = (s[0] + s[1]) + (s[2] + s[3]);
      }
      if (e0 + e < group)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const __half vh = __float2half_rn(x[i]);
          const uint32_t at = ck_block(warp, warp) + ck_in_block(i, cl >> 3) + 2 * (cl & 7);
          *reinterpret_cast<__half*>(sm.img[e].t_hi + at) = vh;
          *reinterpret_cast<__half*>(sm.img[e].t_lo + at) = __float2half_rn(x[i] - __half2float(vh));
        }
      if (p.whole) invert_below(e0);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    if (tid == 0) {
      for (int e = 0; e < 2 && e0 + e < group; ++e)
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(
                         p.images + (int64_t(id) * p.HV + h * group + e0 + e) * CK_IMAGE_BYTES),
                     "r"(smem_addr(&sm.img[e])), "r"(CK_IMAGE_BYTES)
                     : "memory");
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
  }
  if (tid == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

// ---------------------------------------------------------------- chunked form, second kernel, few heads
// Bound by the chain of chunks and the instructions of the one warp on each scheduler: 8192 tokens
// of 32 heads 0.36 ms, 2.8 us a chunk, tensor cores 53 % busy.  (Four warps to 16 rows: 0.52 ms.)
// Four CTAs a head with 32 value rows each; two warps share 16 rows: each
// has half of S's key columns, X and S Q^T are added up through shared memory, both solve for N, and each
// updates its half of S and makes the output of half the tokens.  A fifth warp requests the chunks.
constexpr int CS_WARPS = 4, CS_GROUPS = 2, CS_ROWS = CS_GROUPS * 16, CS_PARTS = 128 / CS_ROWS, CS_THREADS = CS_WARPS * 32 + 32;
constexpr int CS_STAGES = 3;

struct CsStage {  // one chunk
  alignas(1024) uint8_t k[CK_C * 256];
  uint8_t q[CK_C * 256], v[CK_C * 128];
  CkImage img;
};

struct CsSmem {
  CsStage stage[CS_STAGES];
  uint8_t out[CS_WARPS][16 * 48];
  float4 swap[CS_WARPS][12][32];  // a warp's X, and S Q^T of the other's tokens
  uint64_t full[CS_STAGES], empty[CS_STAGES], tail;
};
static_assert(sizeof(CsSmem) + 1024 <= MAX_DYN_SMEM, "one CTA per SM");

__device__ __forceinline__ void plus4(float* x, const float4& y) {
  const float2 a = unpack2(add2(pack2(x[0], x[1]), pack2(y.x, y.y))), b = unpack2(add2(pack2(x[2], x[3]), pack2(y.z, y.w)));
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}

__device__ __forceinline__ void ck_left(const float (*x)[4], uint32_t* hi, uint32_t* lo) {
  split_bf16x2(x[0][0], x[0][1], hi[0], lo[0]);
  split_bf16x2(x[0][2], x[0][3], hi[1], lo[1]);
  split_bf16x2(x[1][0], x[1][1], hi[2], lo[2]);
  split_bf16x2(x[1][2], x[1][3], hi[3], lo[3]);
}

// A power of two that brings a row's largest value (over the four lanes that hold the row) into
// [2^8, 2^9), and its inverse.  N then stays below 2^15: keys are of unit length and beta at most one, so that a token's N is
// at most the sum of 64 R.  At most 2^103: the factors of O, up to 2^7 (a query of zeros), times it and CK_UP stay finite.
__device__ __forceinline__ void ck_row_scale(float top, float& up, float& down) {
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  const int e = min(max(int(__float_as_uint(top) >> 23), 32), 250);
  up = __uint_as_float(uint32_t(262 - e) << 23);
  down = __uint_as_float(uint32_t(e - 8) << 23);
}

// Right operand of block (i, j) of a triangular matrix: both 8-token halves, k of 16
__device__ __forceinline__ void ck_right(uint32_t tri, int i, int j, int lane, uint32_t* b) {
  ldsm_x4(tri + ck_block(i, j) + ck_in_block(((lane >> 4) << 3) + (lane & 7), (lane >> 3) & 1), b);
}

// The n-th sequence from the longest down, so that no long one starts last.  One
// warp, a lane a sequence; larger batches keep their order.
__device__ __forceinline__ int ck_by_length(const PrefillParams& p, int want, int lane) {
  if (p.N == 1 || p.N > 32) return want;
  const int len = lane < p.N ? p.cu[lane + 1] - p.cu[lane] : -1;
  int rank = 0;
  for (int m = 0; m < p.N; ++m) {
    const int other = __shfl_sync(0xffffffffu, len, m);
    rank += other > len || (other == len && m < lane);
  }
  return __ffs(__ballot_sync(0xffffffffu, lane < p.N && rank == want)) - 1;
}

// Column j of blocks of O += N P^T: rows of blocks 0 and 3 where `outer`, of 1 and 2 where `inner`
__device__ __forceinline__ void ck_out_column(float (*O)[4], const uint32_t* nh, const uint32_t* nl, uint32_t ph, uint32_t pl, int j, int lane,
                                              bool outer, bool inner) {
  uint32_t b[4][4], bl[4][4];
#pragma unroll
  for (int i = j; i < 4; ++i)
    if (i == 0 || i == 3 ? outer : inner) {
      ck_right(ph, i, j, lane, b[i]);
      ck_right(pl, i, j, lane, bl[i]);
    }
#pragma unroll
  for (int q = 0; q < 3; ++q)
#pragma unroll
    for (int i = 2 * j; i < 8; ++i)
      if (i < 2 || i > 5 ? outer : inner) {
        const uint32_t* w = (q == 2 ? bl : b)[i >> 1];
        mma_f16(O[i], q == 1 ? nl : nh, w[2 * (i & 1)], w[2 * (i & 1) + 1]);
      }
}

__global__ void __launch_bounds__(CS_THREADS, 1) prefill_scan_kernel(const __grid_constant__ PrefillParams p,
                                                                  const __grid_constant__ CUtensorMap map) {
  extern __shared__ uint8_t raw[];
  CsSmem& sm = *reinterpret_cast<CsSmem*>(raw + (-smem_addr(raw) & 1023u));
  constexpr int PARTS = CS_PARTS, ROWS = CS_ROWS, KT = 8;  // KT: tiles of S of a warp
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int heads = p.HV * PARTS;
  const int n = ck_by_length(p, blockIdx.x / heads, lane);
  const int part = blockIdx.x % heads, hv = part / PARTS, v0 = (part % PARTS) * ROWS;
  const SeqRange r = prefill_seq(p, n);
  if (r.slot < 0) {  // null slot: zero rows
    static_assert(ROWS == 32, "a lane a value");
    for (int t = r.begin + warp; t < r.end; t += CS_THREADS / 32) p.out[t * p.o_st + int64_t(hv) * p.o_sh + v0 + lane] = 0;
    griddep_wait();  // no CTA ends before the first kernel has
    return;
  }
  const bool fresh = p.has_init && !p.has_init[n * p.hi_s];
  if (r.begin == r.end && !fresh) {
    griddep_wait();
    return;
  }
  const int chunks = (r.end - r.begin + CK_C - 1) / CK_C, h = hv / (p.HV / p.H);
  const uint8_t* images = p.images + (int64_t(ck_first(r.begin, n)) * p.HV + hv) * CK_IMAGE_BYTES;

  if (tid == 0) {
    for (int i = 0; i < CS_STAGES; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], CS_WARPS);
    }
    mbar_init(&sm.tail, CS_WARPS);
    fence_mbar_init();
  }
  __syncthreads();
  auto load = [&](int c) {  // one thread
    CsStage& st = sm.stage[c % CS_STAGES];
    uint64_t* bar = &sm.full[c % CS_STAGES];
    const int row = r.begin + c * CK_C;
    mbar_arrive_expect_tx(bar, 2 * CK_C * 256 + CK_C * 128 + CK_IMAGE_BYTES);
    for (int b = 0; b < 2; ++b) {
      ck_tma(smem_addr(st.k) + b * 8192, &map, (p.H + h) * 128 + b * 64, row, bar);
      ck_tma(smem_addr(st.q) + b * 8192, &map, h * 128 + b * 64, row, bar);
    }
    ck_tma(smem_addr(st.v), &map, (2 * p.H + hv) * 128 + (v0 & 64), row, bar);
    bulk_g2s(&st.img, images + int64_t(c) * p.HV * CK_IMAGE_BYTES, CK_IMAGE_BYTES, bar);
  };
  if (warp == CS_WARPS) {
    griddep_wait();  // the images
    if (lane == 0) {
      int c = 0;
      for (; c < chunks; ++c) {
        if (c >= CS_STAGES && !mbar_wait_bounded(&sm.empty[c % CS_STAGES], (c / CS_STAGES - 1) & 1, p.err)) break;
        load(c);
      }
      drain(sm.full, CS_STAGES, c);
    }
    return;
  }
  const int g = lane >> 2, t2 = 2 * (lane & 3);
  const int vr = v0 + (warp % CS_GROUPS) * 16, kh = warp / CS_GROUPS;  // the warp's value rows, its half of the keys
  // S as accumulators: tile n has rows g, g + 8 of the warp's 16 and key columns 8n + t2, + 1
  float* st = p.state + int64_t(r.slot) * p.st_ss + int64_t(hv) * p.st_sh + int64_t(vr + g) * 128 + kh * KT * 8 + t2;
  float S[KT][4];
#pragma unroll
  for (int i = 0; i < KT; ++i) {
    float2 x = make_float2(0.f, 0.f), y = x;
    if (!fresh) {
      x = *reinterpret_cast<const float2*>(st + i * 8);
      y = *reinterpret_cast<const float2*>(st + 8 * 128 + i * 8);
    }
    S[i][0] = x.x, S[i][1] = x.y, S[i][2] = y.x, S[i][3] = y.y;
  }
  const uint32_t os = smem_addr(sm.out[warp]);
  int c = 0;
  bool ok = true;
  for (; c < chunks; ++c) {
    CsStage& tl = sm.stage[c % CS_STAGES];
    const CkImage& im = tl.img;
    const uint32_t ks = smem_addr(tl.k), qs = smem_addr(tl.q), vs = smem_addr(tl.v);
    ok = mbar_wait_bounded(&sm.full[c % CS_STAGES], (c / CS_STAGES) & 1, p.err) && im.made;  // (the pair agrees on it below)
    const int t0 = r.begin + c * CK_C, valid = min(CK_C, r.end - t0);
    if (valid < CK_C) {  // the last chunk
      ck_zero_rows(tl.k, 2, valid, tid, CS_WARPS * 32);
      ck_zero_rows(tl.v, 1, valid, tid, CS_WARPS * 32);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.tail);
      ok = mbar_wait_bounded(&sm.tail, 0, p.err) && ok;
    }
    float X[8][4], O[8][4];
#pragma unroll
    for (int s = 0; s < KT / 2; ++s) {
      uint32_t hi[4], lo[4];
      ck_left(S + 2 * s, hi, lo);
      // products that add to the same tile are kept eight apart: one takes three times as long as it keeps the unit
#pragma unroll
      for (int jj = 0; jj < 4; jj += 2) {
        uint32_t bk[2][4], bq[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t off = ck_at((jj + j) * 16 + ((lane >> 4) << 3) + (lane & 7), kh * KT + s * 2 + ((lane >> 3) & 1));
          ldsm_x4(ks + off, bk[j]);
          ldsm_x4(qs + off, bq[j]);
        }
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (s == 0 && half == 0) {
              mma_bf16_first(X[2 * jj + j], hi, bk[j >> 1][2 * (j & 1)], bk[j >> 1][2 * (j & 1) + 1]);
              mma_bf16_first(O[2 * jj + j], hi, bq[j >> 1][2 * (j & 1)], bq[j >> 1][2 * (j & 1) + 1]);
            } else {
              mma_bf16(X[2 * jj + j], half ? lo : hi, bk[j >> 1][2 * (j & 1)], bk[j >> 1][2 * (j & 1) + 1]);
              mma_bf16(O[2 * jj + j], half ? lo : hi, bq[j >> 1][2 * (j & 1)], bq[j >> 1][2 * (j & 1) + 1]);
            }
          }
      }
    }
    {
      // the other half's X of all tokens and S Q^T of the tokens this warp writes out: blocks 0 and 3, or 1 and 2
#pragma unroll
      for (int j = 0; j < 8; ++j) sm.swap[warp][j][lane] = make_float4(X[j][0], X[j][1], X[j][2], X[j][3]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int mine = j < 2 ? j : j + 4, other = j + 2;  // tiles of blocks 0 and 3, 1 and 2
        sm.swap[warp][8 + j][lane] = kh ? make_float4(O[mine][0], O[mine][1], O[mine][2], O[mine][3])
                                        : make_float4(O[other][0], O[other][1], O[other][2], O[other][3]);
      }
      const int peer = warp ^ CS_GROUPS;
      // the first of a pair's barriers also tells whether either's wait gave up: none is left waiting for the other
      ok = !bar_or(2 + warp % CS_GROUPS, 64, !ok);
      if (!ok) break;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float4 y = sm.swap[peer][j][lane];
        plus4(X[j], y);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4 y = sm.swap[peer][8 + j][lane];
        // kh 0 keeps blocks 0 and 3, kh 1 blocks 1 and 2; the other two are not used again
        plus4(O[j < 2 ? j : j + 4], y);
        plus4(O[j + 2], y);
      }
      bar_sync(2 + warp % CS_GROUPS, 64);  // read before the next chunk's overwrite it
    }
    // R = beta V^T - (beta e^G rk) X
    float top0 = 0.f, top1 = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t w[4];  // tokens 16j + t2 (+1), rows g and g + 8; tokens 16j + 8 + t2
      ldsm_x4_t(vs + swz<128>(j * 16 + ((lane >> 4) << 3) + (lane & 7), ((vr & 63) >> 3) + ((lane >> 3) & 1)), w);
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int tok = j * 16 + hf * 8 + t2;
        // (im.cx holds -beta e^G rk)
        const uint64_t be = pair_at(&im.beta[tok]), cx = pair_at(&im.cx[tok]);
        const float2 v0f = bf16x2_to_f2(w[2 * hf]), v1f = bf16x2_to_f2(w[2 * hf + 1]);
        float* x = X[2 * j + hf];
        const float2 r0 = unpack2(fma2(pack2(x[0], x[1]), cx, mul2(be, pack2(v0f.x, v0f.y))));
        const float2 r1 = unpack2(fma2(pack2(x[2], x[3]), cx, mul2(be, pack2(v1f.x, v1f.y))));
        x[0] = r0.x, x[1] = r0.y, x[2] = r1.x, x[3] = r1.y;
        top0 = fmaxf(top0, fmaxf(fabsf(x[0]), fabsf(x[1])));
        top1 = fmaxf(top1, fmaxf(fabsf(x[2]), fabsf(x[3])));
      }
    }
    // rows to at most 2^9, here CK_UP times them: what the blocks of A take off is of that size
    // The row of O is scaled alike.  Where next to nothing is written (beta of zero) and S is not small, that must not
    // overflow: R then counts as 2^-96 of O at least, far less than what float32 keeps of S beside it.
    if (__any_sync(0xffffffffu, fminf(top0, top1) < 0x1p-60f)) {
      float o0 = 0.f, o1 = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 cq = unpack2(pair_at(&im.cq[j * 8 + t2]));
        o0 = fmaxf(o0, fmaxf(fabsf(O[j][0] * cq.x), fabsf(O[j][1] * cq.y)));
        o1 = fmaxf(o1, fmaxf(fabsf(O[j][2] * cq.x), fabsf(O[j][3] * cq.y)));
      }
      top0 = fmaxf(top0, o0 * 0x1p-96f), top1 = fmaxf(top1, o1 * 0x1p-96f);
    }
    float up0, down0, up1, down1;
    ck_row_scale(top0, up0, down0);
    ck_row_scale(top0, up0, down0);
    ck_row_scale(top1, up1, down1);
    up0 *= CK_UP, up1 *= CK_UP;
    const uint64_t up0_2 = pack2(up0, up0), up1_2 = pack2(up1, up1), back_2 = pack2(CK_DOWN, CK_DOWN);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      scale2(X[j], up0_2);
      scale2(X[j] + 2, up1_2);
      const uint64_t cq = pair_at(&im.cq[j * 8 + t2]);
      scale2(O[j], mul2(cq, up0_2));
      scale2(O[j] + 2, mul2(cq, up1_2));
    }
    const uint32_t th = smem_addr(im.t_hi), tlo = smem_addr(im.t_lo), ph = smem_addr(im.p_hi), pl = smem_addr(im.p_lo);
    float N[8][4];
    uint32_t nh[4][4], nl[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // column j of blocks: T_jj, then -A_ij below it
      uint32_t b[4][4], bl[4][4], rh[4], rl[4];
#pragma unroll
      for (int i = j; i < 4; ++i) {
        ck_right(th, i, j, lane, b[i]);
        ck_right(tlo, i, j, lane, bl[i]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) scale2(X[2 * j + i], back_2), scale2(X[2 * j + i] + 2, back_2);
      ck_left_f16(X + 2 * j, rh, rl);
#pragma unroll
      for (int q = 0; q < 3; ++q)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (q == 0)
            mma_f16_first(N[2 * j + i], rh, b[j][2 * i], b[j][2 * i + 1]);
          else
            mma_f16(N[2 * j + i], q == 1 ? rl : rh, (q == 2 ? bl : b)[j][2 * i], (q == 2 ? bl : b)[j][2 * i + 1]);
#pragma unroll
      for (int i = 0; i < 2; ++i) scale2(N[2 * j + i], back_2), scale2(N[2 * j + i] + 2, back_2);
      ck_left_f16(N + 2 * j, nh[j], nl[j]);
#pragma unroll
      for (int q = 0; q < 3; ++q)
#pragma unroll
        for (int i = 2 * j + 2; i < 8; ++i) {
          const uint32_t* w = (q == 2 ? bl : b)[i >> 1];
          mma_f16(X[i], q == 1 ? nl[j] : nh[j], w[2 * (i & 1)], w[2 * (i & 1) + 1]);
        }
    }
    const uint64_t total = pack2(im.total, im.total), down0_2 = pack2(down0, down0), down1_2 = pack2(down1, down1);
#pragma unroll
    for (int i = 0; i < KT; ++i) {
      scale2(S[i], total);
      scale2(S[i] + 2, total);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t hi[4], lo[4], rest[4];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const uint64_t cs = pair_at(&im.cs[j * 16 + hf * 8 + t2]);
        float* x = N[2 * j + hf];
        scale2(x, mul2(cs, down0_2));
        scale2(x + 2, mul2(cs, down1_2));
        split3_bf16x2(x[0], x[1], hi[2 * hf], lo[2 * hf], rest[2 * hf]);
        split3_bf16x2(x[2], x[3], hi[2 * hf + 1], lo[2 * hf + 1], rest[2 * hf + 1]);
      }
#pragma unroll
      for (int ii = 0; ii < KT / 2; ii += 4) {
        uint32_t b[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) ldsm_x4_t(ks + ck_at(j * 16 + (lane & 15), kh * KT + (ii + i) * 2 + (lane >> 4)), b[i]);
#pragma unroll
        for (int q = 0; q < 3; ++q)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            mma_bf16(S[2 * ii + i], q == 0 ? hi : (q == 1 ? lo : rest), b[i >> 1][2 * (i & 1)], b[i >> 1][2 * (i & 1) + 1]);
      }
    }
    // O += N P^T
#pragma unroll
    for (int j = 0; j < 4; ++j) ck_out_column(O, nh[j], nl[j], ph, pl, j, lane, kh == 0, kh == 1);
    __syncwarp();
    if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(&sm.empty[c % CS_STAGES])) : "memory");
    down0 *= CK_DOWN, down1 *= CK_DOWN;
    // O^T to token rows, 16 tokens at a time through the warp's own rows (48 bytes apart: no bank twice)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (kh != (j == 1 || j == 2)) continue;
      __syncwarp();
      stsm_x4_t(os + (((lane >> 4) << 3) + (lane & 7)) * 48 + ((lane >> 3) & 1) * 16, cvt_bf16x2(O[2 * j][0] * down0, O[2 * j][1] * down0),
                cvt_bf16x2(O[2 * j][2] * down1, O[2 * j][3] * down1), cvt_bf16x2(O[2 * j + 1][0] * down0, O[2 * j + 1][1] * down0),
                cvt_bf16x2(O[2 * j + 1][2] * down1, O[2 * j + 1][3] * down1));
      __syncwarp();
      const int row = j * 16 + (lane >> 1);
      if (row < valid)
        *reinterpret_cast<uint4*>(p.out + int64_t(t0 + row) * p.o_st + int64_t(hv) * p.o_sh + vr + (lane & 1) * 8) =
            *reinterpret_cast<const uint4*>(sm.out[warp] + (lane >> 1) * 48 + (lane & 1) * 16);
    }
  }
  if (!ok) return;  // a wait gave up, here or in the first kernel (the error word says so): the state stays
#pragma unroll
  for (int i = 0; i < KT; ++i) {
    *reinterpret_cast<float2*>(st + i * 8) = make_float2(S[i][0], S[i][1]);
    *reinterpret_cast<float2*>(st + 8 * 128 + i * 8) = make_float2(S[i][2], S[i][3]);
  }
}

// ---------------------------------------------------------------- chunked form, second kernel on tcgen05
// One CTA a sequence and value head: the 128 value rows are the lanes of tensor memory.  Eight warps, two to a
// quarter of the lanes, have half of the columns of a thread's row each (of S's keys, of the chunk's tokens); a ninth
// issues the products, a tenth requests the chunks.  A chunk, as a chain:
//   warps: S -> its two parts          | products: X = S K^T and S Q^T
//   warps: R, near 2^8, as two parts   | N = R T^T
//   warps: weighted N as three parts   | S += it times K
// and beside it N as two parts, N P^T, and the output of the chunk before.
// 3.4 us a chunk (all 128 rows on warp-level tiles: 7.2 us); 12 prompts of up to 2047 tokens, 32 heads: 0.12 ms of
// 0.17.  Bound by the 56 products of a chunk, in four groups one after another (the tensor cores are busy 28 % of the time:
// their A operands come from tensor memory, beside the warps' loads and stores there), and the conversions between.  Slower were: sixteen warps; the output
// taken out before X or after R; P T from the first kernel, which saves the N P^T products, was even (3.3 us a chunk,
// 13 us more for the images).
struct CtStage {  // one chunk
  alignas(1024) uint8_t kq[2 * 16384];  // 64 columns of K and of Q, then the other 64: one right operand of 128 rows
  uint8_t v[CK_C * 256];                // V, then the output
  CkImage img;
};

struct CtSmem {
  CtStage stage[CS_STAGES];
  float top[2][128];
  uint64_t full[CS_STAGES], empty[CS_STAGES];
  uint64_t s_ready, x_done, r_ready, n_done, w_ready, u_done, f_ready, o_done;
  uint64_t top_ready[4], out_ready[2], tail_ready;  // (waits that give up: a barrier would wait for a warp that has given up)
  int abort;
  uint32_t tmem;
};
static_assert(sizeof(CtSmem) + 1024 <= MAX_DYN_SMEM, "one CTA per SM");
constexpr int CT_WARPS = 8, CT_THREADS = (CT_WARPS + 2) * 32;
// tensor memory columns: S; its two bf16 parts, later the three of the weighted N; X = S K^T, later the two f16 parts of R;
// S Q^T; N, later N P^T; the two f16 parts of N
constexpr int CT_S = 0, CT_PARTS = 128, CT_X = 256, CT_Q = 320, CT_N = 384, CT_NF = 448;

__global__ void __launch_bounds__(CT_THREADS, 1) prefill_scan_tc_kernel(const __grid_constant__ PrefillParams p,
                                                                        const __grid_constant__ CUtensorMap map) {
  extern __shared__ uint8_t raw[];
  CtSmem& sm = *reinterpret_cast<CtSmem*>(raw + (-smem_addr(raw) & 1023u));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = ck_by_length(p, blockIdx.x / p.HV, lane), hv = blockIdx.x % p.HV, h = hv / (p.HV / p.H);
  const SeqRange r = prefill_seq(p, n);
  if (r.slot < 0) {  // null slot: zero rows
    for (int t = r.begin + warp; t < r.end; t += CT_THREADS / 32)
      *reinterpret_cast<uint2*>(p.out + t * p.o_st + int64_t(hv) * p.o_sh + lane * 4) = make_uint2(0, 0);
    griddep_wait();  // no CTA ends before the first kernel has
    return;
  }
  const bool fresh = p.has_init && !p.has_init[n * p.hi_s];
  if (r.begin == r.end && !fresh) {
    griddep_wait();
    return;
  }
  const int chunks = (r.end - r.begin + CK_C - 1) / CK_C;
  if (warp == CT_WARPS) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&sm.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else if (tid == 0) {
    for (int i = 0; i < CS_STAGES; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], CT_WARPS + 1);
    }
    mbar_init(&sm.s_ready, CT_WARPS);
    mbar_init(&sm.r_ready, CT_WARPS);
    mbar_init(&sm.w_ready, CT_WARPS);
    mbar_init(&sm.f_ready, CT_WARPS);
    for (int i = 0; i < 2; ++i) mbar_init(&sm.out_ready[i], CT_WARPS / 2);
    mbar_init(&sm.x_done, 1);
    mbar_init(&sm.n_done, 1);
    mbar_init(&sm.o_done, 1);
    mbar_init(&sm.u_done, 1);
    for (int i = 0; i < 4; ++i) mbar_init(&sm.top_ready[i], 2);
    mbar_init(&sm.tail_ready, CT_WARPS);
    sm.abort = 0;
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  const WarpWait wait{p.err, &sm.abort};
  auto full = [&](int c) { return wait(&sm.full[c % CS_STAGES], (c / CS_STAGES) & 1); };
  bool ok = true;

  if (warp == CT_WARPS + 1) {
    // ------------------------------------------------------------ load warp
    griddep_wait();  // the images
    const uint8_t* images = p.images + (int64_t(ck_first(r.begin, n)) * p.HV + hv) * CK_IMAGE_BYTES;
    int c = 0;
    for (; c < chunks; ++c) {
      if (c >= CS_STAGES) ok = wait(&sm.empty[c % CS_STAGES], (c / CS_STAGES - 1) & 1);
      if (!ok) break;
      if (lane == 0) {
        CtStage& st = sm.stage[c % CS_STAGES];
        uint64_t* bar = &sm.full[c % CS_STAGES];
        const int row = r.begin + c * CK_C;
        mbar_arrive_expect_tx(bar, 3 * CK_C * 256 + CK_IMAGE_BYTES);
        for (int b = 0; b < 2; ++b) {
          ck_tma(smem_addr(st.kq) + b * 16384, &map, (p.H + h) * 128 + b * 64, row, bar);
          ck_tma(smem_addr(st.kq) + b * 16384 + 8192, &map, h * 128 + b * 64, row, bar);
          ck_tma(smem_addr(st.v) + b * 8192, &map, (2 * p.H + hv) * 128 + b * 64, row, bar);
        }
        bulk_g2s(&st.img, images + int64_t(c) * p.HV * CK_IMAGE_BYTES, CK_IMAGE_BYTES, bar);
      }
      __syncwarp();
    }
    drain(sm.full, CS_STAGES, c);
  } else if (warp == CT_WARPS) {
    // ------------------------------------------------------------ matrix warp
    for (int c = 0; ok && c < chunks; ++c) {
      CtStage& st = sm.stage[c % CS_STAGES];
      const uint32_t lk = smem_addr(st.kq) >> 4;
      ok = full(c) && wait(&sm.s_ready, c & 1);
      if (!ok) break;
      tc_fence_after();
      if (tc_elect()) {  // S [K^T Q^T]
#pragma unroll
        for (int i = 0; i < 16; ++i)
          tc_mma_ts(tmem + CT_X, tmem + CT_PARTS + i * 8, tc_low_k() + lk + ((i >> 2) & 1) * 1024 + (i & 3) * 2, tc_idesc(2 * CK_C, false), i > 0);
        tc_commit(&sm.x_done);
      }
      __syncwarp();
      // [.., 64] += left [.., 64] in two parts times a triangular matrix in two parts, transposed
      auto triangle = [&](int to, int left, const uint8_t* hi, const uint8_t* lo) {
#pragma unroll
        for (int q = 0; q < 3; ++q) {
          const uint32_t right = tc_low_k() + (smem_addr(q == 2 ? lo : hi) >> 4), from = tmem + left + (q == 1 ? 32 : 0);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            tc_mma_ts<TC_HIGH_32>(tmem + to + 16 * j, from + 8 * j, right + ck_block(j, j) / 16, tc_idesc_f16(CK_C - 16 * j), q + j > 0);
        }
      };
      ok = wait(&sm.r_ready, c & 1);
      if (!ok) break;
      tc_fence_after();
      if (tc_elect()) {
        triangle(CT_N, CT_X, st.img.t_hi, st.img.t_lo);
        tc_commit(&sm.n_done);
      }
      __syncwarp();
      ok = wait(&sm.w_ready, c & 1);
      if (!ok) break;
      tc_fence_after();
      if (tc_elect()) {
#pragma unroll
        for (int i = 0; i < 12; ++i)  // S += weighted N K
          tc_mma_ts(tmem + CT_S, tmem + CT_PARTS + i * 8, tc_low_mn(16384) + lk + (i & 3) * 128, tc_idesc(128, true), 1);
        tc_commit(&sm.u_done);
      }
      __syncwarp();
      ok = wait(&sm.f_ready, c & 1);
      if (!ok) break;
      tc_fence_after();
      if (tc_elect()) {
        triangle(CT_N, CT_NF, st.img.p_hi, st.img.p_lo);
        tc_commit(&sm.o_done);
        tc_commit(&sm.empty[c % CS_STAGES]);
      }
      __syncwarp();
    }
    if (!ok) {  // tensor-core work in flight ends before its memory is given back
      const uint64_t t = globaltimer_ns();
      while (globaltimer_ns() - t < 1000000) {
      }
    }
  } else {
    // ------------------------------------------------------------ a thread a value row
    const int quarter = warp & 3, half = warp >> 2, row = quarter * 32 + lane;
    const uint32_t mem = tmem + (uint32_t(quarter) << 21);
    float* state = p.state + int64_t(r.slot) * p.st_ss + int64_t(hv) * p.st_sh + int64_t(row) * 128 + half * 64;
#pragma unroll 1
    for (int i = 0; i < 64; i += 16) {
      uint32_t w[16];
#pragma unroll
      for (int k = 0; k < 16; k += 4) {
        const uint4 x = fresh ? make_uint4(0, 0, 0, 0) : *reinterpret_cast<const uint4*>(state + i + k);
        w[k] = x.x, w[k + 1] = x.y, w[k + 2] = x.z, w[k + 3] = x.w;
      }
      tc_st16(mem + CT_S + half * 64 + i, w);
    }
    tc_wait_st();
    auto announce = [&](uint64_t* bar) {
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    const int tok = half * 32;  // the thread's tokens of a chunk
    float down = 0.f, sq[32];   // the row's scale (back from N, CK_UP times it), S q of its tokens: kept until the chunk's output is written
    // The output of chunk c over V, then to memory in whole rows.  Called after the next chunk's products have begun.
    auto finish = [&](int c) {
      CtStage& st = sm.stage[c % CS_STAGES];
      const int t0 = r.begin + c * CK_C, valid = min(CK_C, r.end - t0);
      if (!wait(&sm.o_done, c & 1)) return false;
      tc_fence_after();
      float y[32];
      tc_ld32(mem + CT_N + tok, y);
      tc_wait_ld();
      uint8_t* v = st.v + (row >> 6) * 8192 + (row & 7) * 2;
#pragma unroll
      for (int k = 0; k < 32; k += 2) {
        const uint32_t w = cvt_bf16x2(fmaf(y[k], down, sq[k]), fmaf(y[k + 1], down, sq[k + 1]));
        *reinterpret_cast<uint16_t*>(v + swz<128>(tok + k, (row & 63) >> 3)) = uint16_t(w);
        *reinterpret_cast<uint16_t*>(v + swz<128>(tok + k + 1, (row & 63) >> 3)) = uint16_t(w >> 16);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.out_ready[half]);
      if (!wait(&sm.out_ready[half], c & 1)) return false;
      uint16_t* to = p.out + int64_t(t0) * p.o_st + int64_t(hv) * p.o_sh;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = tok + i * 8 + (tid & 127) / 16, j = tid & 15;
        if (t < valid) *reinterpret_cast<uint4*>(to + t * p.o_st + j * 8) = *reinterpret_cast<const uint4*>(st.v + ck_at(t, j));
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before TMA writes the V of a later chunk there
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.empty[c % CS_STAGES]);
      return true;
    };
    for (int c = 0; c < chunks; ++c) {
      CtStage& st = sm.stage[c % CS_STAGES];
      const CkImage& im = st.img;
      const int t0 = r.begin + c * CK_C, valid = min(CK_C, r.end - t0);
      ok = full(c);
      if (ok && !im.made) ok = false, sm.abort = 1;
      if (ok && c) ok = wait(&sm.u_done, (c - 1) & 1);
      if (!ok) break;
      tc_fence_after();
      if (valid < CK_C) {  // the last chunk
        ck_zero_rows(st.kq, 1, valid, tid, CT_WARPS * 32);
        ck_zero_rows(st.kq + 16384, 1, valid, tid, CT_WARPS * 32);
        ck_zero_rows(st.v, 2, valid, tid, CT_WARPS * 32);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.tail_ready);
        ok = wait(&sm.tail_ready, 0);
        if (!ok) break;
      }
      // S as two parts for the products, and decayed for what is added to it
      {
        const uint64_t total = pack2(im.total, im.total);
#pragma unroll
        for (int i = 0; i < 64; i += 32) {
          float s[32];
          tc_ld32(mem + CT_S + half * 64 + i, s);
          tc_wait_ld();
          uint32_t hi[16], lo[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            split_bf16x2(s[2 * k], s[2 * k + 1], hi[k], lo[k]);
            scale2(s + 2 * k, total);
          }
          tc_st16(mem + CT_PARTS + half * 32 + i / 2, hi);
          tc_st16(mem + CT_PARTS + 64 + half * 32 + i / 2, lo);
          tc_st16(mem + CT_S + half * 64 + i, reinterpret_cast<uint32_t*>(s));
          tc_st16(mem + CT_S + half * 64 + i + 16, reinterpret_cast<uint32_t*>(s) + 16);
        }
      }
      announce(&sm.s_ready);
      if (c) {
        ok = finish(c - 1);
        if (!ok) break;
      }
      // R = beta V^T - (beta e^G rk) X
      {
        float x[32];
        uint64_t bv[16];
        const uint8_t* v = st.v + (row >> 6) * 8192 + (row & 7) * 2;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const float v0 = bf16_to_f(*reinterpret_cast<const uint16_t*>(v + swz<128>(tok + 2 * k, (row & 63) >> 3)));
          const float v1 = bf16_to_f(*reinterpret_cast<const uint16_t*>(v + swz<128>(tok + 2 * k + 1, (row & 63) >> 3)));
          bv[k] = mul2(pair_at(&im.beta[tok + 2 * k]), pack2(v0, v1));
        }
        ok = wait(&sm.x_done, c & 1);
        if (!ok) break;
        tc_fence_after();
        tc_ld32(mem + CT_X + tok, x);
        tc_wait_ld();
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          const float2 y = unpack2(fma2(pack2(x[k], x[k + 1]), pair_at(&im.cx[tok + k]), bv[k / 2]));
          x[k] = y.x, x[k + 1] = y.y;
          top = fmaxf(top, fmaxf(fabsf(y.x), fabsf(y.y)));
        }
        // the row near 2^8 for f16, by the largest of all 64 tokens
        sm.top[half][row] = top;
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.top_ready[quarter]);  // both warps have read X then, too
        ok = wait(&sm.top_ready[quarter], c & 1);
        if (!ok) break;
        top = fmaxf(top, sm.top[half ^ 1][row]);
        // (as ck_row_scale)
        const int e = min(max(int(__float_as_uint(top) >> 23), 32), 250);
        const float up = __uint_as_float(uint32_t(262 - e) << 23);
        down = __uint_as_float(uint32_t(e - 8) << 23) * CK_DOWN;
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) split_f16x2(x[2 * k] * up, x[2 * k + 1] * up, hi[k], lo[k]);
        tc_st16(mem + CT_X + half * 16, hi);
        tc_st16(mem + CT_X + 32 + half * 16, lo);
      }
      announce(&sm.r_ready);
      // what is added to S first: the next chunk waits for it
      tc_ld32(mem + CT_Q + tok, sq);
      tc_wait_ld();
#pragma unroll
      for (int k = 0; k < 32; k += 2) scale2(sq + k, pair_at(&im.cq[tok + k]));
      {
        const uint64_t down2 = pack2(down, down);
        ok = wait(&sm.n_done, c & 1);
        if (!ok) break;
        tc_fence_after();
        float x[32];
        tc_ld32(mem + CT_N + tok, x);
        tc_wait_ld();
        uint32_t hi[16], lo[16], rest[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          float w[2] = {x[2 * k], x[2 * k + 1]};
          scale2(w, mul2(pair_at(&im.cs[tok + 2 * k]), down2));
          split3_bf16x2(w[0], w[1], hi[k], lo[k], rest[k]);
        }
        tc_st16(mem + CT_PARTS + half * 16, hi);
        tc_st16(mem + CT_PARTS + 32 + half * 16, lo);
        tc_st16(mem + CT_PARTS + 64 + half * 16, rest);
        announce(&sm.w_ready);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          scale2(x + 2 * k, pack2(CK_DOWN, CK_DOWN));
          split_f16x2(x[2 * k], x[2 * k + 1], hi[k], lo[k]);
        }
        tc_st16(mem + CT_NF + half * 16, hi);
        tc_st16(mem + CT_NF + 32 + half * 16, lo);
        announce(&sm.f_ready);
      }
    }
    if (ok && chunks) ok = finish(chunks - 1);
    if (ok && chunks) ok = wait(&sm.u_done, (chunks - 1) & 1);
    if (ok) {  // (a wait that gave up, here or in the first kernel, leaves the state as it was)
      tc_fence_after();
#pragma unroll 1
      for (int i = 0; i < 64; i += 32) {
        float s[32];
        tc_ld32(mem + CT_S + half * 64 + i, s);
        tc_wait_ld();
#pragma unroll
        for (int k = 0; k < 32; k += 4) *reinterpret_cast<float4*>(state + i + k) = make_float4(s[k], s[k + 1], s[k + 2], s[k + 3]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == CT_WARPS) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// May be set up while the first kernel's last CTAs run: they wait for the images (griddep_wait).
template <class K>
cudaError_t launch_scan(K kern, DynSmemCache& cache, int ctas, int threads, int smem, const PrefillParams& p, const CUtensorMap& map,
                        cudaStream_t stream) {
  const cudaError_t e = ensure_dyn_smem(reinterpret_cast<const void*>(kern), smem + 1024, cache);
  return e != cudaSuccess ? e : launch_behind(kern, dim3(unsigned(int64_t(p.N) * p.HV * ctas)), threads, smem + 1024, stream, p, map);
}

}  // namespace

cudaError_t launch_prefill_chunk(PrefillParams p, int64_t longest, cudaStream_t stream) {
  CUtensorMap map;
  // boxes of 64 columns x 64 tokens of mixed_qkv
  const uint64_t dims[2] = {uint64_t(2 * p.H + p.HV) * 128, uint64_t(p.T)};
  const uint64_t strides[1] = {uint64_t(p.mx_s) * 2};
  const uint32_t box[2] = {64, CK_C};
  cudaError_t e = encode_bf16_map(&map, p.mixed, 2, dims, strides, box);
  if (e != cudaSuccess) return e;
  static DynSmemCache cache;
  constexpr int bytes = sizeof(CdSmem) + 1024;
  e = ensure_dyn_smem(reinterpret_cast<const void*>(prefill_derive_kernel), bytes, cache);
  if (e != cudaSuccess) return e;
  const int64_t ids = int64_t(p.T) / CK_C + p.N;
  // A head's 128 value rows on one multiprocessor (3.4 us a chunk), or on four, 32 each with their key columns halved
  // (2.8 us, 12 us of multiprocessor time a head's chunk).  What takes longest is the chunks of all sequences, spread
  // over the machine, or those of the longest one after another.  32 heads: 8 prompts of 2048 tokens 0.34 / 0.72 ms,
  // 64 of 64 tokens 0.18 / 0.31 ms, 2 of 2048 tokens 0.15 / 0.21 ms; 1 of 8192 tokens 0.50 / 0.40 ms.
  const int64_t chain = (longest + CK_C - 1) / CK_C, all = ids * p.HV / multiprocessor_count();
  p.whole = std::max(all * 120, chain * 28) > std::max(all, chain) * 34;
  prefill_derive_kernel<<<dim3(unsigned(ids * p.H)), CD_THREADS, bytes, stream>>>(p, map);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  static DynSmemCache tc_cache, scan_cache;
  return p.whole ? launch_scan(prefill_scan_tc_kernel, tc_cache, 1, CT_THREADS, sizeof(CtSmem), p, map, stream)
                 : launch_scan(prefill_scan_kernel, scan_cache, CS_PARTS, CS_THREADS, sizeof(CsSmem), p, map, stream);
}

// The longest sequence as the host knows it, or the mean length
static int64_t longest_of(int64_t tokens, int64_t sequences, int max_seqlen) {
  return max_seqlen > 0 ? std::min<int64_t>(max_seqlen, tokens) : (tokens + sequences - 1) / sequences;
}

// Twenty tokens a sequence token by token / as a chunk, 32 heads: 1 sequence 15 / 15 us, 12 sequences 50 / 50 us, 64 sequences
// 216 / 215 us, 128 sequences 415 / 419 us.
static bool prefill_chunked(int64_t tokens, int64_t sequences, int max_seqlen) { return longest_of(tokens, sequences, max_seqlen) > 20; }

int64_t prefill_workspace_bytes(int64_t tokens, int64_t sequences, int64_t value_heads, int max_seqlen) {
  if (sequences <= 0 || tokens <= 0 || !prefill_chunked(tokens, sequences, max_seqlen)) return 0;
  return (tokens / CK_C + sequences) * value_heads * CK_IMAGE_BYTES;
}

cudaError_t launch_prefill(const PrefillParams& p, int max_seqlen, cudaStream_t stream) {
  if (p.T == 0 || !prefill_chunked(p.T, p.N, max_seqlen)) return launch_prefill_recurrent(p, stream);
  return launch_prefill_chunk(p, longest_of(p.T, p.N, max_seqlen), stream);
}

cudaError_t launch_prefill_recurrent(const PrefillParams& p, cudaStream_t stream) {
  const int64_t blocks = int64_t(p.N) * p.HV * (128 / (RC_ROWS * RC_WARPS));
  prefill_recurrent_kernel<<<dim3(unsigned(blocks)), RC_WARPS * 32, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace gdnr
