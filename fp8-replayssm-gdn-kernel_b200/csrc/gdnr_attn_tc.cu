// Paged attention of sequences with many rows, on tcgen05.
//
// A CTA walks its share of the batch's (row tile, key tile) pairs.  NQ streams of 128 rows (one
// where D = 256, whose accumulator takes half of tensor memory) share the keys and
// values, which TMA brings page by page into a ring of tiles:
//   load warp      query rows of each unit, keys and values of tile 0, 1, ...
//   matrix warp    S = Q K^T into tensor memory; O += P V with P from tensor memory
//   softmax warps  four a stream, a thread a row: S -> registers, maximum, exponentials, their sum,
//                  P as bf16 over S
// While one stream's softmax runs, the tensor cores work for the other (or, with one
// stream, on the next tile's S).  The reference maximum of a row only moves when the row's maximum
// has grown by more than 2^8 (p <= 2^8 keeps bf16's relative precision); only then O is rescaled.
//
// 2048 tokens over 32768 keys, 16 / 2 heads of 128: 416 us, 1.28 PFLOP/s in bursts of a hundred calls, 480 to 490 us, 1.1 PFLOP/s
// in runs of seconds, under the power cap (heads of 256 over 16384 keys: 458 and 527 us, 1.13 and 0.98 PFLOP/s).  A stream's
// softmax (1 us a tile) and its two products (0.6 us) alternate, as tensor memory has no room for a second S; the
// other stream fills most of the gaps.  Slower were: tiles of 64 keys with two buffers of S each, P announced by
// halves, some of the exponentials by a polynomial.
#include "gdnr_attn.cuh"
#include "gdnr_tc.cuh"

#include <algorithm>

namespace gdnr {

namespace {

template <int D>
struct TcCfg {
  static constexpr int NQ = D == 256 ? 1 : 2;
  static constexpr int BN = D == 256 ? 64 : 128;
  static constexpr int BM = 128 * NQ;
  static constexpr int ATOMS = D / 64;                  // 64-element (128-byte) column blocks
  static constexpr int Q_BYTES = 128 * D * 2;           // a stream
  static constexpr int KV_BYTES = BN * D * 2;           // a tile of keys or of values
  static constexpr int RING = D == 256 ? 5 : (D == 128 ? 5 : 8);
  static constexpr int SOFTMAX_WARPS = 4 * NQ;
  // two streams: whole groups of four warps, and registers are handed from the last one (two of its warps have no
  // role) to the softmax warps, whose rows of S live in them: 256 x 200 + 128 x 104 <= 384 x 168, what the block is
  // launched with
  static constexpr int THREADS = 32 * (SOFTMAX_WARPS + (NQ == 2 ? 4 : 2));
  static constexpr int SOFTMAX_REGS = 200, OTHER_REGS = 104;
  static constexpr int SMEM = NQ * Q_BYTES + RING * KV_BYTES + 1024;
  // tensor memory columns: two buffers of S (P lies over the first half of its S), then O
  static constexpr int S_COLS = BN, O_COL = 256;
  static constexpr int OVER = D == 256 ? 4 : 2;  // a unit's beginning and end, 4 to 5 us, in tiles of 0.9 or 2.3 us
  static_assert(SMEM + 512 <= 227 * 1024, "one CTA per SM");
};

__device__ __forceinline__ void tc_tma3(uint32_t dst, const CUtensorMap* map, int c, int h, int token, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(c), "r"(h), "r"(token), "r"(smem_addr(bar))
      : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <bool DO, int REGS>
__device__ __forceinline__ void tc_regs_dec() {
  if constexpr (DO) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS));
}

struct TcBars {
  uint64_t kv_full[8], kv_empty[8];
  uint64_t q_full[2];   // the stream's query rows are in shared memory
  uint64_t q_free[2];   // matrix warp -> load warp: the stream's last Q K^T of a unit is complete
  uint64_t s_full[2];   // matrix warp -> softmax warps: S of the buffer is complete
  uint64_t p_full[2];   // softmax warps -> matrix warp: P of the buffer is written (and O rescaled)
  uint64_t o_full;      // one stream: PV of a key tile is complete (what O must wait for before it is rescaled)
  uint64_t done[2];     // matrix warp -> softmax warps: the stream's last PV of a unit is complete
  int abort;
  uint32_t tmem;
  int64_t places[12];
};

template <int D>
__global__ void __launch_bounds__(TcCfg<D>::THREADS, 1)
    attn_tc_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                   const __grid_constant__ CUtensorMap qmap, const AtRows of, const int q_tma) {
  using C = TcCfg<D>;
  using T = AtTile<C::BM, C::BN, C::OVER>;
  constexpr int NQ = C::NQ, BN = C::BN, BM = C::BM;
  extern __shared__ uint8_t raw[];
  __shared__ TcBars bars;
  const uint32_t base = (smem_addr(raw) + 1023u) & ~1023u, kv_base = base + NQ * C::Q_BYTES;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  float* const ws_o = p.ws + int64_t(blockIdx.x) * 2 * BM * (D + 2);
  int* const meta = reinterpret_cast<int*>(p.ws + int64_t(gridDim.x) * 2 * BM * (D + 2)) + blockIdx.x * AT_META;

  if (of.lo > 0) griddep_launch();  // the few-row kernel takes over a multiprocessor when this CTA ends
  constexpr int WARPS = C::THREADS / 32;
  const int64_t places = warp_places<T>(p, of, warp, WARPS, lane);
  if (lane == 0) bars.places[warp] = places;
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&bars.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else if (tid == 64) {
    for (int i = 0; i < C::RING; ++i) {
      mbar_init(&bars.kv_full[i], 1);
      mbar_init(&bars.kv_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.q_full[i], q_tma ? 1 : 4);
      mbar_init(&bars.q_free[i], 1);
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_full[i], 4);
      mbar_init(&bars.done[i], 1);
    }
    mbar_init(&bars.o_full, 1);
    bars.abort = 0;
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem;
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) total += bars.places[w];
  const Share share = share_of<T>(total, blockIdx.x, gridDim.x);
  const WarpWait wait{p.err, &bars.abort};
  Unit u;
  u.n = p.N;
  if (share.begin < share.end) {
    u = find_unit<T>(p, of, share.begin, bars.places, WARPS, lane);
    if (tid == 0) write_meta<T>(meta, share, u, total, gridDim.x);
  } else if (tid == 0) {
    meta[0] = -1;
  }

  // key tiles [t0, t1) of the unit are this share's; stream q sees the first seen(q) tiles of the unit
  auto seen = [&](int q) {
    const int rows = u.rt * BM + (q + 1) * 128;
    if (u.rt * BM + q * 128 >= u.s.m * p.G) return 0;
    return max(0, (keys_seen(p, u.s, rows) + BN - 1) / BN);
  };

  if (warp == C::SOFTMAX_WARPS + 1) {
    // ------------------------------------------------------------ load warp
    tc_regs_dec<C::NQ == 2, C::OTHER_REGS>();
    uint32_t slot = 0, nq[2] = {0, 0};  // tiles and query tiles requested so far
    bool ok = true;
    for (int64_t at = share.begin; ok && at < share.end; next_unit<T>(p, of, u), at = u.begin) {
      const Tiles part_of = tiles_of<T>(share, u);
      const int t0 = part_of.begin;
      int t1 = part_of.end;
      if (t1 <= t0) continue;
      int most = seen(0);
      if (NQ > 1) most = max(most, seen(1));
      t1 = min(t1, most);
      const int32_t* table = p.table + int64_t(u.n) * p.tb_s;
      for (int q = 0; q_tma && q < NQ && ok; ++q) {
        if (min(t1, seen(q)) <= t0) continue;
        if (nq[q]) ok = wait(&bars.q_free[q], (nq[q] - 1) & 1);
        if (!ok) break;
        ++nq[q];
        if (lane == 0) mbar_arrive_expect_tx(&bars.q_full[q], C::Q_BYTES);
        __syncwarp();
        // rows past the sequence's end are another's: their results are not written
        if (lane < C::ATOMS)
          tc_tma3(base + q * C::Q_BYTES + lane * 16384, &qmap, lane * 64, u.h * p.G, u.s.q0 + token_of(p, u.rt * BM + q * 128), &bars.q_full[q]);
      }
      for (int t = t0; ok && t < t1; ++t) {
        const KvBox b = kv_box<BN, C::ATOMS>(p, u, table, t, lane);
        for (int kv = 0; kv < 2; ++kv, ++slot) {
          const uint32_t s = slot % C::RING;
          if (slot >= C::RING) ok = wait(&bars.kv_empty[s], (slot / C::RING - 1) & 1);
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&bars.kv_full[s], C::KV_BYTES);
          __syncwarp();
          if (b.live)
            kv_tma(kv_base + s * C::KV_BYTES + b.to, kv ? &vmap : &kmap, b.col, u.h, b.off, b.page, &bars.kv_full[s]);
        }
      }
    }
    for (int q = 0; q < NQ; ++q) drain(&bars.q_full[q], 1, nq[q]);
    drain(bars.kv_full, C::RING, slot);
  } else if (warp == C::SOFTMAX_WARPS) {
    // ------------------------------------------------------------ matrix warp
    tc_regs_dec<C::NQ == 2, C::OTHER_REGS>();
    uint32_t slot = 0, nq[2] = {0, 0}, np[2] = {0, 0};  // tiles consumed; phases of q_full, p_full
    constexpr uint32_t QK = tc_idesc(BN, false), PV = tc_idesc(D, true);
    bool ok = true;
    auto kv_wait = [&](uint32_t k) { return wait(&bars.kv_full[k % C::RING], (k / C::RING) & 1); };
    auto kv_addr = [&](uint32_t k) { return kv_base + (k % C::RING) * C::KV_BYTES; };
    auto score = [&](int q, int buf, uint32_t k, bool last) {  // S[buf] = Q_q K^T
      const uint32_t lq = tc_low_k() + ((base + q * C::Q_BYTES) >> 4), lk = tc_low_k() + (kv_addr(k) >> 4), to = tmem + buf * C::S_COLS;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        tc_mma_ss(to, lq + (i >> 2) * 1024 + (i & 3) * 2, lk + (i >> 2) * (BN * 8) + (i & 3) * 2, QK, i > 0);
      tc_commit(&bars.s_full[buf]);
      if (last) tc_commit(&bars.q_free[q]);
    };
    auto weigh = [&](int q, int buf, uint32_t k, bool first, bool last) {  // O_q += P[buf] V
      const uint32_t lv = tc_low_mn(BN * 128) + (kv_addr(k) >> 4), from = tmem + buf * C::S_COLS;
#pragma unroll
      for (int i = 0; i < BN / 16; ++i)
        tc_mma_ts(tmem + C::O_COL + q * D, from + i * 8, lv + i * 128, PV, !first || i > 0);
      if (NQ == 1) tc_commit(&bars.o_full);
      if (last) tc_commit(&bars.done[q]);
    };
    for (int64_t at = share.begin; ok && at < share.end; next_unit<T>(p, of, u), at = u.begin) {
      const Tiles part_of = tiles_of<T>(share, u);
      const int t0 = part_of.begin, t1 = part_of.end;
      if (t1 <= t0) continue;
      int end[2] = {min(t1, seen(0)), NQ > 1 ? min(t1, seen(1)) : 0};
      const int last = max(end[0], end[1]);
      if (last <= t0) continue;
      for (int q = 0; q < NQ && ok; ++q)
        if (end[q] > t0) ok = wait(&bars.q_full[q], nq[q]++ & 1);
      // tile t: keys in slot k0 + 2 (t - t0), values in the next one
      const uint32_t k0 = slot;
      // the last page may end inside the tile: what its rows past the end hold (it may be NaN) must not meet a weight of zero
      auto clean = [&](int t, uint32_t k) {
        const int from = u.s.kv - t * BN;
        if (from >= BN) return;
        for (int i = lane; i < (BN - from) * C::ATOMS * 8; i += 32) {
          const int row = from + i / (C::ATOMS * 8), j = i % (C::ATOMS * 8);
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(kv_addr(k) + (j >> 3) * (BN * 128) + row * 128 + (j & 7) * 16), "r"(0)
                       : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
      };
      auto free_slot = [&](uint32_t k) {
        if (tc_elect()) tc_commit(&bars.kv_empty[k % C::RING]);
      };
      if constexpr (NQ == 2) {
        // S0(t), S1(t); then for each stream P(t) V(t) and S(t + 1)
        if (ok) ok = kv_wait(k0);
        if (ok && tc_elect())
          for (int q = 0; q < 2; ++q)
            if (end[q] > t0) score(q, q, k0, t0 + 1 == end[q]);
        free_slot(k0);
        for (int t = t0; t < last && ok; ++t) {
          const uint32_t kk = k0 + 2 * (t + 1 - t0), kv = k0 + 2 * (t - t0) + 1;
          ok = kv_wait(kv);
          if (!ok) break;
          clean(t, kv);
          bool have_k = false;
          for (int q = 0; q < 2 && ok; ++q) {
            if (t >= end[q]) continue;
            ok = wait(&bars.p_full[q], np[q]++ & 1);
            if (!ok) break;
            tc_fence_after();
            if (tc_elect()) weigh(q, q, kv, t == t0, t + 1 == end[q]);
            if (t + 1 < end[q]) {
              if (!have_k) ok = kv_wait(kk), have_k = true;
              if (!ok) break;
              if (tc_elect()) score(q, q, kk, t + 2 == end[q]);
            }
            __syncwarp();
          }
          free_slot(kv);
          if (t + 1 < last) free_slot(kk);
        }
      } else {
        // S(t + 1) is issued before P(t) V(t), into the other buffer
        if (ok) ok = kv_wait(k0);
        if (ok && tc_elect()) score(0, t0 & 1, k0, t0 + 1 == last);
        free_slot(k0);
        for (int t = t0; t < last && ok; ++t) {
          const uint32_t kk = k0 + 2 * (t + 1 - t0), kv = k0 + 2 * (t - t0) + 1;
          if (t + 1 < last) {
            ok = kv_wait(kk);
            if (!ok) break;
            if (tc_elect()) score(0, (t + 1) & 1, kk, t + 2 == last);
            __syncwarp();
            free_slot(kk);
          }
          ok = kv_wait(kv);
          if (!ok) break;
          clean(t, kv);
          ok = wait(&bars.p_full[t & 1], np[t & 1]++ & 1);
          if (!ok) break;
          tc_fence_after();
          if (tc_elect()) weigh(0, t & 1, kv, t == t0, t + 1 == last);
          __syncwarp();
          free_slot(kv);
        }
      }
      slot = k0 + 2 * (last - t0);
    }
    if (!ok) {  // tensor-core work in flight ends before its memory is given back
      const uint64_t t = globaltimer_ns();
      while (globaltimer_ns() - t < 1000000) {
      }
    }
  } else if (warp < C::SOFTMAX_WARPS) {
    // ------------------------------------------------------------ softmax warps
    if constexpr (NQ == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::SOFTMAX_REGS));
    const int q = NQ > 1 ? warp >> 2 : 0, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = uint32_t(warp & 3) << 21;  // the warp's tensor memory lanes (bits 16..)
    const uint32_t q_smem = base + q * C::Q_BYTES, o_mem = tmem + lanes + C::O_COL + q * D;
    const float sl2 = p.scale * LOG2E;
    uint32_t ns[2] = {0, 0}, no = 0, nd = 0;  // phases of s_full, o_full, done
    bool ok = true;
    for (int64_t at = share.begin; ok && at < share.end; next_unit<T>(p, of, u), at = u.begin) {
      const Tiles part_of = tiles_of<T>(share, u);
      const int t0 = part_of.begin, t1 = part_of.end;
      if (t1 <= t0) continue;
      const int end = min(t1, seen(q));
      const int row = u.rt * BM + q * 128 + r;  // row of the sequence
      const bool live = row < u.s.m * p.G;
      const int lim = live ? min(u.s.kv - 1, u.s.kv - u.s.m + token_of(p, row)) : -1;  // last key the row sees
      if (tid == 0) report_unit(p, u);
      float mx = -INFINITY, sum = 0.f;
      if (end > t0 && !q_tma) {
        // D / 8 lanes copy a row, eight loads in flight; rows past the sequence's are zeros
        constexpr int CH = D / 8;
#pragma unroll 1
        for (int i0 = lane; i0 < 32 * CH; i0 += 256) {
          uint4 x[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int i = i0 + j * 32, rr = (warp & 3) * 32 + i / CH, srow = u.rt * BM + q * 128 + rr, tk = token_of(p, srow);
            x[j] = make_uint4(0, 0, 0, 0);
            if (srow < u.s.m * p.G)
              x[j] = *reinterpret_cast<const uint4*>(p.q + int64_t(u.s.q0 + tk) * p.q_st + int64_t(u.h * p.G + srow - tk * p.G) * p.q_sh +
                                                     i % CH * 8);
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int i = i0 + j * 32, rr = (warp & 3) * 32 + i / CH, c = i % CH;
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(q_smem + (c >> 3) * 16384 + swz<128>(rr, c & 7)), "r"(x[j].x),
                         "r"(x[j].y), "r"(x[j].z), "r"(x[j].w)
                         : "memory");
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.q_full[q]);
      }
      const int warp_lim = __reduce_min_sync(0xffffffffu, lim);
      for (int t = t0; t < end; ++t) {
        const int buf = NQ > 1 ? q : t & 1;
        ok = wait(&bars.s_full[buf], ns[buf]++ & 1);
        if (!ok) break;
        tc_fence_after();
        const uint32_t s_mem = tmem + lanes + buf * C::S_COLS;
        float s[BN];
#pragma unroll
        for (int i = 0; i < BN / 32; ++i) tc_ld32(s_mem + i * 32, s + i * 32);
        tc_wait_ld();
        if (warp_lim < t * BN + BN - 1) {  // some row of the warp does not see the whole tile
          const int left = lim - t * BN;
#pragma unroll
          for (int i = 0; i < BN; ++i) s[i] = i <= left ? s[i] : -INFINITY;
        }
        float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int i = 4; i + 8 <= BN; i += 8)
#pragma unroll
          for (int j = 0; j < 4; ++j) top[j] = max3(top[j], s[i + j], s[i + 4 + j]);
#pragma unroll
        for (int j = 0; j < 4; ++j) top[j] = fmaxf(top[j], s[BN - 4 + j]);
        const float tm = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * sl2;
        if (t == t0) {
          mx = tm;
        } else if (__any_sync(0xffffffffu, tm > mx + 8.0f)) {
          // O is at rest once the previous tile's PV is; its phase cannot pass before this tile's P
          if constexpr (NQ == 1) {
            ok = wait(&bars.o_full, (no - 1) & 1);
            if (!ok) break;
          }
          tc_fence_after();
          const bool grow = tm > mx + 8.0f;
          const float f = grow ? ex2_approx(mx - tm) : 1.0f;
          if (grow) mx = tm;
          sum *= f;
#pragma unroll 1
          for (int i = 0; i < D; i += 16) {
            float o[16];
            tc_ld16(o_mem + i, o);
            tc_wait_ld();
            uint32_t w[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = __float_as_uint(o[j] * f);
            tc_st16(o_mem + i, w);
          }
        }
        const float b = mx == -INFINITY ? 0.f : mx;  // a row that has seen no key yet
        uint64_t part[2] = {0, 0};  // pairs of sums
        const uint64_t sl2_2 = pack2(sl2, sl2), nb2 = pack2(-b, -b);
#pragma unroll
        for (int i = 0; i < BN / 32; ++i) {
          uint32_t w[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float2 e = unpack2(fma2(pack2(s[i * 32 + 2 * j], s[i * 32 + 2 * j + 1]), sl2_2, nb2));
            const float x = ex2_approx(e.x), y = ex2_approx(e.y);
            part[j & 1] = add2(part[j & 1], pack2(x, y));
            // weights are rounded to bf16 for the tensor cores; their sum is taken before that
            w[j] = cvt_bf16x2(x, y);
          }
          tc_st16(s_mem + i * 16, w);
        }
        tc_wait_st();
        const float2 add = unpack2(add2(part[0], part[1]));
        sum += add.x + add.y;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.p_full[buf]);
        ++no;
      }
      if (!ok) break;
      const bool any = end > t0;
      if (any) {
        ok = wait(&bars.done[q], nd++ & 1);
        if (!ok) break;
        tc_fence_after();
      }
      const bool whole = t0 == 0 && t1 == u.tiles;
      const float inv = sum > 0.f ? 1.0f / sum : 0.f;
      uint16_t* dst = live ? p.out + out_at(p, u, row) : nullptr;
      float* part = ws_o + (t0 > 0 ? 0 : 1) * BM * (D + 2) + q * 128 + r;  // columns of BM rows
#pragma unroll 1
      for (int i = 0; i < D; i += 32) {
        float o[32];
        if (any) {
          tc_ld32(o_mem + i, o);
          tc_wait_ld();
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = 0.f;
        }
        if (live && whole) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<uint4*>(dst + i + j * 8) =
                make_uint4(cvt_bf16x2(o[8 * j] * inv, o[8 * j + 1] * inv), cvt_bf16x2(o[8 * j + 2] * inv, o[8 * j + 3] * inv),
                           cvt_bf16x2(o[8 * j + 4] * inv, o[8 * j + 5] * inv), cvt_bf16x2(o[8 * j + 6] * inv, o[8 * j + 7] * inv));
        } else if (live) {
#pragma unroll
          for (int j = 0; j < 32; ++j) part[(i + j) * BM] = o[j];
        }
        __syncwarp();
      }
      if (live) {
        if (whole)
          write_lse(p, u.s, u.h, row, mx, sum);
        else
          part[D * BM] = mx, part[(D + 1) * BM] = sum;
      }
      tc_fence_before();  // O has been read before the next unit's first P is announced
      __syncwarp();
    }
  } else {
    tc_regs_dec<C::NQ == 2, C::OTHER_REGS>();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

template <int D>
cudaError_t run_tc(const AttnParams& p, const AtRows& of, cudaStream_t stream) {
  using C = TcCfg<D>;
  CUtensorMap maps[2];
  cudaError_t e = encode_kv_maps(p, C::BN, maps);
  if (e != cudaSuccess) return e;
  static DynSmemCache cache;
  auto kern = attn_tc_kernel<D>;
  e = ensure_dyn_smem(reinterpret_cast<const void*>(kern), C::SMEM, cache);
  if (e != cudaSuccess) return e;
  const int ctas = multiprocessor_count();
  // query rows by TMA where a tile is whole tokens: boxes of 64 elements x G heads x 128 / G tokens
  CUtensorMap qmap = maps[0];
  const int q_tma = 128 % p.G == 0 && p.q_st > 0 && p.q_sh > 0 && p.q_st % 8 == 0 && p.q_sh % 8 == 0;
  if (q_tma) {
    const uint64_t dims[3] = {uint64_t(D), uint64_t(p.Hq), uint64_t(p.T)};
    const uint64_t strides[2] = {uint64_t(p.q_sh) * 2, uint64_t(p.q_st) * 2};
    const uint32_t box[3] = {64, uint32_t(p.G), uint32_t(128 / p.G)};
    e = encode_bf16_map(&qmap, p.q, 3, dims, strides, box);
    if (e != cudaSuccess) return e;
  }
  kern<<<ctas, C::THREADS, C::SMEM, stream>>>(p, maps[0], maps[1], qmap, of, q_tma);
  return cudaGetLastError();
}

}  // namespace

int64_t attn_tc_floats(int head_dim) {
  return int64_t(multiprocessor_count()) * (2 * attn_tc_rows(head_dim) * (head_dim + 2) + AT_META);
}

// Scores that grow with the dot product: the maximum is taken before the scale
bool attn_tc_takes(const AttnParams& p) { return p.scale > 0.f && kv_tma_takes(p); }

cudaError_t launch_attn_tc(const AttnParams& p, int lo, cudaStream_t stream) {
  const AtRows of{lo, INT32_MAX};
  if (p.D == 64) return run_tc<64>(p, of, stream);
  if (p.D == 128) return run_tc<128>(p, of, stream);
  return run_tc<256>(p, of, stream);
}

}  // namespace gdnr
