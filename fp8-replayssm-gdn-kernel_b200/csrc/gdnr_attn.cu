// Causal attention of each sequence's new tokens over its paged cache (gdnr_paged_attention).
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i.k_j - max),  j <= kv - m + i
//
// for the m new tokens i of a sequence of kv tokens.  The G = Hq/Hk query heads of a key
// head are rows of one tile (row r of a sequence: token r / G, head r % G), so a key
// or value read from memory serves all of them.
#include "gdnr_attn.cuh"

#include <algorithm>

namespace gdnr {

namespace {

constexpr int AT_BN = 64;  // keys of a tile
constexpr int AT_MAX_CTAS_PER_SM = 2;

// ---------------------------------------------------------------- kernel
// WM x WN warps: WM groups of 16 rows, each tile's keys cut over WN warps that keep
// their own running maximum and sum and are joined at the unit's end.
template <int D, int WM, int WN, int STAGES>
struct AtCfg {
  static constexpr int BM = 16 * WM;
  static constexpr int THREADS = 32 * WM * WN;
  static constexpr int ROWB = D * 2;
  static constexpr int TILE = AT_BN * ROWB;
  static constexpr int Q_BYTES = BM * ROWB;
  static constexpr int JOIN = WN > 1 ? WN * 16 * (D + 4) * 4 : 0;
  static constexpr int SMEM = Q_BYTES + STAGES * 2 * TILE;
  static_assert(JOIN <= STAGES * 2 * TILE, "the join reuses the stages");
};

template <int D, int WM, int WN, int STAGES>
__global__ void __launch_bounds__(32 * WM * WN) attn_kernel(const __grid_constant__ AttnParams p, const AtRows of) {
  using C = AtCfg<D, WM, WN, STAGES>;
  using T = AtTile<C::BM, AT_BN, 1>;
  constexpr int BM = C::BM, ROWB = C::ROWB, CH = ROWB / 16, NT = AT_BN / WN / 8;  // NT: 8-key tiles of a warp
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int WARPS = WM * WN;
  __shared__ int64_t sh_places[WARPS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wm = warp / WN, wn = warp % WN;
  const uint32_t q_s = smem_addr(smem), kv_s = q_s + C::Q_BYTES;
  float* const ws_o = p.ws + int64_t(blockIdx.x) * 2 * BM * (D + 2);
  int* const meta = reinterpret_cast<int*>(p.ws + int64_t(gridDim.x) * 2 * BM * (D + 2)) + blockIdx.x * AT_META;

  const int64_t places = warp_places<T>(p, of, warp, WARPS, lane);
  if (lane == 0) sh_places[warp] = places;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) total += sh_places[w];
  const Share share = share_of<T>(total, blockIdx.x, gridDim.x);
  if (share.begin >= share.end) {
    if (tid == 0) meta[0] = -1;
    return;
  }
  Unit u = find_unit<T>(p, of, share.begin, sh_places, WARPS, lane);
  if (tid == 0) write_meta<T>(meta, share, u, total, gridDim.x);
  const float sl2 = p.scale * LOG2E;
  for (int64_t at = share.begin; at < share.end; next_unit<T>(p, of, u), at = u.begin) {
    const Tiles part_of = tiles_of<T>(share, u);
    const int t0 = part_of.begin, t1 = part_of.end;
    if (t1 <= t0) continue;
    const int rows = u.s.m * p.G - u.rt * BM;  // rows of the sequence from this tile on
    const int row_base = u.rt * BM;
    const int32_t* table = p.table + int64_t(u.n) * p.tb_s;
    if (tid == 0) report_unit(p, u);
    // query rows of the tile; rows beyond the sequence's are zeros
    for (int i = tid; i < BM * CH; i += C::THREADS) {
      const int r = i / CH, c = i % CH;
      const bool ok = r < rows;
      const int rr = row_base + (ok ? r : 0), tk = token_of(p, rr);
      cp_async16_zfill(q_s + swz<ROWB>(r, c), p.q + int64_t(u.s.q0 + tk) * p.q_st + int64_t(u.h * p.G + rr - tk * p.G) * p.q_sh + c * 8,
                       ok ? 16 : 0);
    }
    auto load_tile = [&](int t, int stage) {
      const uint32_t ks = kv_s + stage * 2 * C::TILE, vs = ks + C::TILE;
      for (int i = tid; i < AT_BN * CH; i += C::THREADS) {
        const int r = i / CH, c = i % CH;
        const int tok = t * AT_BN + r;
        const uint16_t *ksrc = p.k, *vsrc = p.v;
        uint32_t bytes = 0;
        // keys past the sequence's end are never read: what a page holds there may be anything
        if (tok < u.s.kv) {
          const int pi = p.page_shift >= 0 ? tok >> p.page_shift : tok / p.page_size;
          const int off = tok - pi * p.page_size;
          const int page = table[pi];
          if (page >= 0 && page < p.pages) {
            ksrc += int64_t(page) * p.k_sp + int64_t(off) * p.k_st + int64_t(u.h) * p.k_sh + c * 8;
            vsrc += int64_t(page) * p.v_sp + int64_t(off) * p.v_st + int64_t(u.h) * p.v_sh + c * 8;
            bytes = 16;
          } else {
            atomicOr(p.err, GDNR_DEVERR_BAD_SLOT);
          }
        }
        cp_async16_zfill(ks + swz<ROWB>(r, c), ksrc, bytes);
        cp_async16_zfill(vs + swz<ROWB>(r, c), vsrc, bytes);
      }
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) {
      if (t0 + s < t1) load_tile(t0 + s, s);
      cp_async_commit();
    }
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
    // last key each of this thread's two rows sees
    int lim[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = row_base + wm * 16 + (lane >> 2) + 8 * j;
      lim[j] = r < u.s.m * p.G ? min(u.s.kv - 1, u.s.kv - u.s.m + token_of(p, r)) : -1;
    }
    for (int t = t0; t < t1; ++t) {
      const int i = t - t0;
      cp_async_wait<STAGES - 2>();
      __syncthreads();
      if (t + STAGES - 1 < t1) load_tile(t + STAGES - 1, (i + STAGES - 1) % STAGES);
      cp_async_commit();
      const uint32_t ks = kv_s + (i % STAGES) * 2 * C::TILE, vs = ks + C::TILE;
      float s[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t a[4];
        ldsm_x4(q_s + swz<ROWB>(wm * 16 + (lane & 15), kk * 2 + (lane >> 4)), a);
#pragma unroll
        for (int j = 0; j < NT / 2; ++j) {
          uint32_t b[4];
          ldsm_x4(ks + swz<ROWB>(wn * (AT_BN / WN) + j * 16 + ((lane >> 4) << 3) + (lane & 7), kk * 2 + ((lane >> 3) & 1)), b);
          mma16816_bf16(s[2 * j], a, b[0], b[1]);
          mma16816_bf16(s[2 * j + 1], a, b[2], b[3]);
        }
      }
      const int key0 = t * AT_BN + wn * (AT_BN / WN) + 2 * (lane & 3);
      float tm[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // a comparison, not an added bias: whatever a masked score is, it leaves no trace
          s[j][e] = key0 + j * 8 + (e & 1) <= lim[e >> 1] ? s[j][e] * sl2 : -INFINITY;
          tm[e >> 1] = fmaxf(tm[e >> 1], s[j][e]);
        }
      float corr[2], base[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        tm[j] = fmaxf(tm[j], __shfl_xor_sync(0xffffffffu, tm[j], 1));
        tm[j] = fmaxf(tm[j], __shfl_xor_sync(0xffffffffu, tm[j], 2));
        const float nm = fmaxf(mx[j], tm[j]);
        base[j] = nm == -INFINITY ? 0.f : nm;  // a row that has seen no key yet
        corr[j] = ex2_approx(mx[j] - base[j]);
        mx[j] = nm;
        sum[j] *= corr[j];
      }
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[j][e] = ex2_approx(s[j][e] - base[e >> 1]);
          sum[e >> 1] += s[j][e];
        }
#pragma unroll
      for (int j = 0; j < D / 8; ++j) {
        o[j][0] *= corr[0];
        o[j][1] *= corr[0];
        o[j][2] *= corr[1];
        o[j][3] *= corr[1];
      }
#pragma unroll
      for (int kk = 0; kk < NT / 2; ++kk) {
        // weights are rounded to bf16 for the tensor cores; their sum is taken before that
        uint32_t a[4] = {pack_bf16x2(s[2 * kk][0], s[2 * kk][1]), pack_bf16x2(s[2 * kk][2], s[2 * kk][3]),
                         pack_bf16x2(s[2 * kk + 1][0], s[2 * kk + 1][1]), pack_bf16x2(s[2 * kk + 1][2], s[2 * kk + 1][3])};
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          uint32_t b[4];
          ldsm_x4_t(vs + swz<ROWB>(wn * (AT_BN / WN) + kk * 16 + (lane & 15), j * 2 + (lane >> 4)), b);
          mma16816_bf16(o[2 * j], a, b[0], b[1]);
          mma16816_bf16(o[2 * j + 1], a, b[2], b[3]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 1);
      sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 2);
    }
    cp_async_wait<0>();
    __syncthreads();  // every warp is done with the tiles and the query rows
    const bool whole = t0 == 0 && t1 == u.tiles;
    // a share that begins inside a unit leaves its part in slot 0, one that only ends inside in slot 1
    float* part = ws_o + (t0 > 0 ? 0 : 1) * BM * (D + 2);
    if constexpr (WN == 1) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = wm * 16 + (lane >> 2) + 8 * j;
        if (r >= rows) continue;
        if (whole) {
          const float inv = sum[j] > 0.f ? 1.0f / sum[j] : 0.f;
          uint16_t* dst = p.out + out_at(p, u, row_base + r) + 2 * (lane & 3);
#pragma unroll
          for (int c = 0; c < D / 8; ++c)
            *reinterpret_cast<uint32_t*>(dst + c * 8) = pack_bf16x2(o[c][2 * j] * inv, o[c][2 * j + 1] * inv);
          if ((lane & 3) == 0) write_lse(p, u.s, u.h, row_base + r, mx[j], sum[j]);
        } else {
          float* dst = part + r * (D + 2);
#pragma unroll
          for (int c = 0; c < D / 8; ++c)
            *reinterpret_cast<float2*>(dst + c * 8 + 2 * (lane & 3)) = make_float2(o[c][2 * j], o[c][2 * j + 1]);
          if ((lane & 3) == 0) dst[D] = mx[j], dst[D + 1] = sum[j];
        }
      }
    } else {
      // join the WN warps' parts of the 16 rows through shared memory
      static_assert(WM == 1 || WN == 1, "one of the two");
      float* js = reinterpret_cast<float*>(smem + C::Q_BYTES);
      constexpr int LD = D + 4;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float* dst = js + (wn * 16 + (lane >> 2) + 8 * j) * LD;
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
          *reinterpret_cast<float2*>(dst + c * 8 + 2 * (lane & 3)) = make_float2(o[c][2 * j], o[c][2 * j + 1]);
        if ((lane & 3) == 0) dst[D] = mx[j], dst[D + 1] = sum[j];
      }
      __syncthreads();
      for (int r = warp; r < 16 && r < rows; r += WM * WN) {
        float m = -INFINITY, f[WN], l = 0.f;
#pragma unroll
        for (int w = 0; w < WN; ++w) m = fmaxf(m, js[(w * 16 + r) * LD + D]);
        const float b = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int w = 0; w < WN; ++w) {
          f[w] = ex2_approx(js[(w * 16 + r) * LD + D] - b);
          l += f[w] * js[(w * 16 + r) * LD + D + 1];
        }
        const int64_t to = out_at(p, u, row_base + r);
        const float inv = l > 0.f ? 1.0f / l : 0.f;
        for (int c = lane * 2; c < D; c += 64) {
          float2 x = make_float2(0.f, 0.f);
#pragma unroll
          for (int w = 0; w < WN; ++w) {
            const float2 y = *reinterpret_cast<const float2*>(js + (w * 16 + r) * LD + c);
            x.x += f[w] * y.x;
            x.y += f[w] * y.y;
          }
          if (whole)
            *reinterpret_cast<uint32_t*>(p.out + to + c) = pack_bf16x2(x.x * inv, x.y * inv);
          else
            *reinterpret_cast<float2*>(part + r * (D + 2) + c) = x;
        }
        if (lane == 0) {
          if (!whole)
            part[r * (D + 2) + D] = m, part[r * (D + 2) + D + 1] = l;
          else
            write_lse(p, u.s, u.h, row_base + r, m, l);
        }
      }
      __syncthreads();  // the next unit's tiles overwrite the join
    }
  }
}

// ---------------------------------------------------------------- kernel, pages by TMA
// The same tiles and the same split, with the keys and values requested by a warp of its own page by page
// (attn_kernel's threads spend four fifths of their instructions on copying: 64 sequences of 4 k keys took
// 135 us; here 86 us, 5.9 TB/s).  Needs page sizes that are multiples of 8.
template <int D, int WM, int WN, int STAGES>
struct AsCfg {
  static constexpr int BM = 16 * WM, CONSUMERS = 32 * WM * WN, THREADS = CONSUMERS + 32;
  static constexpr int ROWB = D * 2, ATOMS = D / 64, TILE = AT_BN * ROWB, Q_BYTES = BM * ROWB;
  // the first kilobyte: AsShared; the stages begin at the second, a multiple of 1024 bytes (two CTAs of 115,712 bytes
  // are what a multiprocessor holds: there is no room to align by hand)
  static constexpr int SMEM = 1024 + STAGES * 2 * TILE + Q_BYTES;
  static_assert(WN == 1 || WM * WN * 16 * D * 4 <= 2 * TILE, "the join uses the last tile's stage");
};

struct AsShared {
  uint64_t full[8], empty[8];
  int64_t places[5];
  int abort;
  float ml[4][16][2];  // maximum and sum of the rows of each warp's keys
};
static_assert(sizeof(AsShared) <= 1024, "the first kilobyte");

template <int D, int WM, int WN, int STAGES>
__global__ void __launch_bounds__(32 * WM * WN + 32)
    attn_stream_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                       const AtRows of) {
  using C = AsCfg<D, WM, WN, STAGES>;
  using T = AtTile<C::BM, AT_BN, 1>;
  constexpr int BM = C::BM, ROWB = C::ROWB, CH = ROWB / 16, NT = AT_BN / WN / 8;  // NT: 8-key tiles of a warp
  extern __shared__ __align__(1024) uint8_t raw[];
  AsShared& sh = *reinterpret_cast<AsShared*>(raw);
  uint64_t *const full = sh.full, *const empty = sh.empty;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t kv_s = smem_addr(raw) + 1024, q_s = kv_s + STAGES * 2 * C::TILE;
  float* const ws_o = p.ws + int64_t(blockIdx.x) * 2 * BM * (D + 2);
  int* const meta = reinterpret_cast<int*>(p.ws + int64_t(gridDim.x) * 2 * BM * (D + 2)) + blockIdx.x * AT_META;
  if (kv_s & 1023u) {  // the swizzled tiles would not be where the products look for them
    if (tid == 0) {
      atomicOr(p.err, GDNR_DEVERR_LAYOUT);
      meta[0] = -1;  // nothing to join
    }
    griddep_wait();
    return;
  }

  constexpr int WARPS = WM * WN + 1;
  static_assert(WARPS == 5, "AsShared::places");
  const int64_t places = warp_places<T>(p, of, warp, WARPS, lane);
  if (lane == 0) sh.places[warp] = places;
  if (tid == 32) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], WM * WN);
    }
    sh.abort = 0;
    fence_mbar_init();
  }
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) total += sh.places[w];
  const Share share = share_of<T>(total, blockIdx.x, gridDim.x);
  if (share.begin >= share.end) {
    if (tid == 0) meta[0] = -1;
    griddep_wait();
    return;
  }
  const WarpWait wait{p.err, &sh.abort};
  Unit u = find_unit<T>(p, of, share.begin, sh.places, WARPS, lane);
  uint32_t k = 0;  // tiles requested or consumed so far
  bool ok = true;

  if (warp == WM * WN) {
    for (int64_t at = share.begin; ok && at < share.end; next_unit<T>(p, of, u), at = u.begin) {
      const Tiles part_of = tiles_of<T>(share, u);
      const int t0 = part_of.begin, t1 = part_of.end;
      if (t1 <= t0) continue;
      const int32_t* table = p.table + int64_t(u.n) * p.tb_s;
      for (int t = t0; t < t1; ++t, ++k) {
        const KvBox b = kv_box<AT_BN, C::ATOMS>(p, u, table, t, lane);
        const uint32_t s = k % STAGES, to = kv_s + s * 2 * C::TILE;
        if (k >= STAGES) ok = wait(&empty[s], (k / STAGES - 1) & 1);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&full[s], 2 * C::TILE);
        __syncwarp();
        if (b.live) {
          kv_tma(to + b.to, &kmap, b.col, u.h, b.off, b.page, &full[s]);
          kv_tma(to + C::TILE + b.to, &vmap, b.col, u.h, b.off, b.page, &full[s]);
        }
      }
    }
    drain(full, STAGES, k);
    // a CTA does not end before the kernel that this one may run beside has: what comes next waits for this one only
    griddep_wait();
    return;
  }

  if (tid == 0) write_meta<T>(meta, share, u, total, gridDim.x);
  const int wm = warp / WN, wn = warp % WN;
  const float sl2 = p.scale * LOG2E;
  for (int64_t at = share.begin; at < share.end; next_unit<T>(p, of, u), at = u.begin) {
    const Tiles part_of = tiles_of<T>(share, u);
    const int t0 = part_of.begin, t1 = part_of.end;
    if (t1 <= t0) continue;
    const int row_base = u.rt * BM, rows = u.s.m * p.G - row_base;  // rows of the sequence from this tile on
    if (tid == 0) report_unit(p, u);
    // query rows of the tile; rows beyond the sequence's are zeros
    for (int i = tid; i < BM * CH; i += C::CONSUMERS) {
      const int r = i / CH, c = i % CH;
      const bool in = r < rows;
      const int rr = row_base + (in ? r : 0), tk = token_of(p, rr);
      cp_async16_zfill(q_s + swz<ROWB>(r, c), p.q + int64_t(u.s.q0 + tk) * p.q_st + int64_t(u.h * p.G + rr - tk * p.G) * p.q_sh + c * 8,
                       in ? 16 : 0);
    }
    cp_async_commit();
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
    int lim[2];  // last key each of this thread's two rows sees
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = row_base + wm * 16 + (lane >> 2) + 8 * j;
      lim[j] = r < u.s.m * p.G ? min(u.s.kv - 1, u.s.kv - u.s.m + token_of(p, r)) : -1;
    }
    const int low = __reduce_min_sync(0xffffffffu, min(lim[0], lim[1]));
    cp_async_wait<0>();
    bar_sync(1, C::CONSUMERS);
    for (int t = t0; t < t1; ++t, ++k) {
      const uint32_t st = k % STAGES, ks = kv_s + st * 2 * C::TILE, vs = ks + C::TILE;
      ok = wait(&full[st], (k / STAGES) & 1);
      if (!ok) break;  // straight to the unit's next barrier
      // the last page may end inside the tile: what its rows past the end hold (it may be NaN) must not meet a weight of zero
      const int from = u.s.kv - t * AT_BN;
      if (from < AT_BN) {
        const int r0 = WN > 1 ? wn * (AT_BN / WN) : 0, r1 = WN > 1 ? r0 + AT_BN / WN : AT_BN;
        const int first = max(from, r0), step = WN > 1 ? 32 : C::CONSUMERS;
        for (int i = WN > 1 ? lane : tid; i < (r1 - first) * CH; i += step) {
          const int r = first + i / CH, c = i % CH;
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(vs + (c >> 3) * (AT_BN * 128) + r * 128 + (c & 7) * 16), "r"(0)
                       : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        if (WN > 1)
          __syncwarp();
        else if (bar_or(1, C::CONSUMERS, false))
          return;
      }
      float s[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t a[4];
        ldsm_x4(q_s + swz<ROWB>(wm * 16 + (lane & 15), kk * 2 + (lane >> 4)), a);
#pragma unroll
        for (int j = 0; j < NT / 2; ++j) {
          uint32_t b[4];
          const int r = wn * (AT_BN / WN) + j * 16 + ((lane >> 4) << 3) + (lane & 7), c = kk * 2 + ((lane >> 3) & 1);
          ldsm_x4(ks + (c >> 3) * (AT_BN * 128) + swz<128>(r, c & 7), b);
          mma_bf16(s[2 * j], a, b[0], b[1]);
          mma_bf16(s[2 * j + 1], a, b[2], b[3]);
        }
      }
      const int key0 = t * AT_BN + wn * (AT_BN / WN) + 2 * (lane & 3);
      if (low < t * AT_BN + AT_BN - 1) {  // some row does not see the whole tile
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            // a comparison, not an added bias: whatever a masked score is, it leaves no trace
            s[j][e] = key0 + j * 8 + (e & 1) <= lim[e >> 1] ? s[j][e] * sl2 : -INFINITY;
      } else {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[j][e] *= sl2;
      }
      float base[2];
      bool grow = false;
      float nm[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float tm = fmaxf(s[0][2 * j], s[0][2 * j + 1]);
#pragma unroll
        for (int i = 1; i < NT; ++i) tm = fmaxf(tm, fmaxf(s[i][2 * j], s[i][2 * j + 1]));
        tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, 1));
        nm[j] = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, 2));
        grow = grow || nm[j] > mx[j] + 8.0f;
      }
      // the reference maximum moves only when a row's has grown by more than 2^8 (weights then keep their
      // relative precision), so that O is rarely rescaled
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float m = fmaxf(mx[j], nm[j]), f = ex2_approx(mx[j] - (m == -INFINITY ? 0.f : m));
          mx[j] = m;
          sum[j] *= f;
#pragma unroll
          for (int i = 0; i < D / 8; ++i) o[i][2 * j] *= f, o[i][2 * j + 1] *= f;
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) base[j] = mx[j] == -INFINITY ? 0.f : mx[j];  // a row that has seen no key yet
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[j][e] = ex2_approx(s[j][e] - base[e >> 1]);
          sum[e >> 1] += s[j][e];
        }
#pragma unroll
      for (int kk = 0; kk < NT / 2; ++kk) {
        // Weights are rounded to bf16 for the tensor cores; their sum is taken before that.  (As two bf16 each, which would leave the
        // output's own rounding only: 64 single tokens 1 to 5 % slower, drafts up to 20 %.)
        const uint32_t a[4] = {cvt_bf16x2(s[2 * kk][0], s[2 * kk][1]), cvt_bf16x2(s[2 * kk][2], s[2 * kk][3]),
                               cvt_bf16x2(s[2 * kk + 1][0], s[2 * kk + 1][1]), cvt_bf16x2(s[2 * kk + 1][2], s[2 * kk + 1][3])};
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          uint32_t b[4];
          const int r = wn * (AT_BN / WN) + kk * 16 + (lane & 15), c = j * 2 + (lane >> 4);
          ldsm_x4_t(vs + (c >> 3) * (AT_BN * 128) + swz<128>(r, c & 7), b);
          mma_bf16(o[2 * j], a, b[0], b[1]);
          mma_bf16(o[2 * j + 1], a, b[2], b[3]);
        }
      }
      __syncwarp();
      if (lane == 0 && (WN == 1 || t + 1 < t1)) mbar_arrive(&empty[st]);  // the join below uses the last one
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 1);
      sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 2);
    }
    // Every warp is done with the query rows and the last tile.  The first barrier that a warp meets after a wait also tells
    // whether any warp's wait gave up: then all leave, none is left at a barrier that another does not come to.
    if (bar_or(1, C::CONSUMERS, !ok)) return;
    const bool whole = t0 == 0 && t1 == u.tiles;
    float* part = ws_o + (t0 > 0 ? 0 : 1) * BM * (D + 2);
    if constexpr (WN == 1) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = wm * 16 + (lane >> 2) + 8 * j;
        if (r >= rows) continue;
        if (whole) {
          const float inv = sum[j] > 0.f ? 1.0f / sum[j] : 0.f;
          uint16_t* dst = p.out + out_at(p, u, row_base + r) + 2 * (lane & 3);
#pragma unroll
          for (int c = 0; c < D / 8; ++c)
            *reinterpret_cast<uint32_t*>(dst + c * 8) = cvt_bf16x2(o[c][2 * j] * inv, o[c][2 * j + 1] * inv);
          if ((lane & 3) == 0) write_lse(p, u.s, u.h, row_base + r, mx[j], sum[j]);
        } else {
          float* dst = part + r * (D + 2);
#pragma unroll
          for (int c = 0; c < D / 8; ++c)
            *reinterpret_cast<float2*>(dst + c * 8 + 2 * (lane & 3)) = make_float2(o[c][2 * j], o[c][2 * j + 1]);
          if ((lane & 3) == 0) dst[D] = mx[j], dst[D + 1] = sum[j];
        }
      }
    } else {
      // join the WN warps' parts of each 16 rows in the last tile's stage, [WM][WN][16][D] floats, columns changed by row
      const uint32_t st = (k - 1) % STAGES;
      float* js = reinterpret_cast<float*>(raw + 1024 + st * 2 * C::TILE);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = (lane >> 2) + 8 * j;
        float* dst = js + (warp * 16 + r) * D;
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
          *reinterpret_cast<float2*>(dst + ((c * 8 + 2 * (lane & 3)) ^ ((r & 7) * 8))) = make_float2(o[c][2 * j], o[c][2 * j + 1]);
        if ((lane & 3) == 0) sh.ml[warp][r][0] = mx[j], sh.ml[warp][r][1] = sum[j];
      }
      bar_sync(1, C::CONSUMERS);
      for (int r = warp; r < BM && r < rows; r += WM * WN) {
        const int w0 = (r >> 4) * WN, r16 = r & 15;  // its warps, its row there
        float m = -INFINITY, f[WN], l = 0.f;
#pragma unroll
        for (int w = 0; w < WN; ++w) m = fmaxf(m, sh.ml[w0 + w][r16][0]);
        const float b = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int w = 0; w < WN; ++w) {
          f[w] = ex2_approx(sh.ml[w0 + w][r16][0] - b);
          l += f[w] * sh.ml[w0 + w][r16][1];
        }
        const int64_t to = out_at(p, u, row_base + r);
        const float inv = l > 0.f ? 1.0f / l : 0.f;
#pragma unroll
        for (int c = lane * 2; c < D; c += 64) {
          float2 x = make_float2(0.f, 0.f);
#pragma unroll
          for (int w = 0; w < WN; ++w) {
            const float2 y = *reinterpret_cast<const float2*>(js + ((w0 + w) * 16 + r16) * D + (c ^ ((r & 7) * 8)));
            x.x += f[w] * y.x;
            x.y += f[w] * y.y;
          }
          if (whole)
            *reinterpret_cast<uint32_t*>(p.out + to + c) = cvt_bf16x2(x.x * inv, x.y * inv);
          else
            *reinterpret_cast<float2*>(part + r * (D + 2) + c) = x;
        }
        if (lane == 0) {
          if (!whole)
            part[r * (D + 2) + D] = m, part[r * (D + 2) + D + 1] = l;
          else
            write_lse(p, u.s, u.h, row_base + r, m, l);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before TMA writes there again
      bar_sync(1, C::CONSUMERS);
      if (lane == 0) mbar_arrive(&empty[st]);
    }
  }
}

// Joins the parts of the units that are cut between shares.  Block (i, y) looks at
// the cut between shares i - 1 and i: where it is the first cut of its unit, the
// block joins ROWS rows of all parts in the order of the shares (a fixed order: the
// result does not depend on which CTA ran when).  The eight warps have a row each, or share one
// row's parts: a unit of few rows may be cut into as many parts as there are shares.
constexpr int AJ_WARPS = 8;

// A kernel's parts, and how many blocks look at a cut.
struct Cuts {
  const float* ws;
  AtRows rows;
  int ctas, ys;
};

template <int D, int BM, int ROWS>
__device__ __forceinline__ void join_rows(const AttnParams& p, const Cuts& of, int i, int y0) {
  constexpr int PER_ROW = AJ_WARPS / ROWS;
  __shared__ float sm[AJ_WARPS][D + 2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  CutUnit cut;
  if (!cut_unit(reinterpret_cast<const int*>(of.ws + int64_t(of.ctas) * 2 * BM * (D + 2)), i, cut)) return;
  const SeqLen s = seq_len(p, cut.n, of.rows);
  const int r = y0 * ROWS + warp / PER_ROW, rr = cut.rt * BM + r;
  const bool live = r < BM && rr < s.m * p.G;
  if (__syncthreads_or(live) == 0) return;
  constexpr int E = D / 32;
  float m = -INFINITY, l = 0.f, x[E];
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = 0.f;
  if (live) {
    const int parts = cut.parts;
    constexpr int AHEAD = 4;
    for (int c0 = warp % PER_ROW; c0 < parts; c0 += PER_ROW * AHEAD) {
      float y[AHEAD][E], pm[AHEAD], pl[AHEAD];
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        const int c = c0 + a * PER_ROW;
        pm[a] = -INFINITY, pl[a] = 0.f;
        const float* src = of.ws + (int64_t(i - 1 + c) * 2 + (c == 0 ? 1 : 0)) * BM * (D + 2) + int64_t(r) * (D + 2);
        if (c < parts) pm[a] = src[D], pl[a] = src[D + 1];
#pragma unroll
        for (int e = 0; e < E; ++e) y[a][e] = c < parts ? src[e * 32 + lane] : 0.f;
      }
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        const float nm = fmaxf(m, pm[a]), b = nm == -INFINITY ? 0.f : nm;
        const float f0 = ex2_approx(m - b), f1 = ex2_approx(pm[a] - b);
        m = nm;
        l = l * f0 + pl[a] * f1;
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = x[e] * f0 + y[a][e] * f1;
      }
    }
  }
  if constexpr (PER_ROW > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) sm[warp][e * 32 + lane] = x[e];
    if (lane == 0) sm[warp][D] = m, sm[warp][D + 1] = l;
    __syncthreads();
    const int w0 = warp / PER_ROW * PER_ROW;
    if (warp != w0) return;
    m = -INFINITY;
#pragma unroll
    for (int w = 0; w < PER_ROW; ++w) m = fmaxf(m, sm[w0 + w][D]);
    const float b = m == -INFINITY ? 0.f : m;
    l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = 0.f;
#pragma unroll
    for (int w = 0; w < PER_ROW; ++w) {
      const float f = ex2_approx(sm[w0 + w][D] - b);
      l += f * sm[w0 + w][D + 1];
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] += f * sm[w0 + w][e * 32 + lane];
    }
  }
  if (!live) return;
  const float inv = l > 0.f ? 1.0f / l : 0.f;
  const int tk = token_of(p, rr);
  uint16_t* dst = p.out + int64_t(s.q0 + tk) * p.o_st + int64_t(cut.h * p.G + rr - tk * p.G) * p.o_sh;
#pragma unroll
  for (int e = 0; e < E; ++e) dst[e * 32 + lane] = f_to_bf16(x[e] * inv);
  if (lane == 0) write_lse(p, s, cut.h, rr, m, l);
}

// The same for parts that lie in columns of BM rows (the tcgen05 kernel's: its threads have a row each).  Block
// (i, y) has 32 rows, a lane each, and AJ_WARPS * COLS columns, COLS a warp.
template <int D, int BM, int COLS, int AHEAD>
__device__ __forceinline__ void join_columns(const AttnParams& p, const Cuts& of, int i, int y0) {
  constexpr int BLOCKS = D / (AJ_WARPS * COLS);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  CutUnit cut;
  if (!cut_unit(reinterpret_cast<const int*>(of.ws + int64_t(of.ctas) * 2 * BM * (D + 2)), i, cut)) return;
  const SeqLen s = seq_len(p, cut.n, of.rows);
  const int col = (y0 % BLOCKS * AJ_WARPS + warp) * COLS, r = y0 / BLOCKS * 32 + lane, rr = cut.rt * BM + r;
  if (rr >= s.m * p.G) return;
  float m = -INFINITY, l = 0.f, x[COLS];
#pragma unroll
  for (int e = 0; e < COLS; ++e) x[e] = 0.f;
  // the next parts are on their way while some are added
  float next[AHEAD][COLS], nm[AHEAD], nl[AHEAD];
  auto request = [&](int c0) {
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int c = c0 + a;
      if (AHEAD > 1 && c >= cut.parts) break;
      const float* src = of.ws + (int64_t(i - 1 + c) * 2 + (c == 0 ? 1 : 0)) * BM * (D + 2) + r;
      nm[a] = src[D * BM], nl[a] = src[(D + 1) * BM];
#pragma unroll
      for (int e = 0; e < COLS; ++e) next[a][e] = src[(col + e) * BM];
    }
  };
  request(0);
  for (int c0 = 0; c0 < cut.parts; c0 += AHEAD) {
    float y[AHEAD][COLS], pm[AHEAD], pl[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      pm[a] = nm[a], pl[a] = nl[a];
#pragma unroll
      for (int e = 0; e < COLS; ++e) y[a][e] = next[a][e];
    }
    if (c0 + AHEAD < cut.parts) request(c0 + AHEAD);
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      if (AHEAD > 1 && c0 + a >= cut.parts) break;
      const float top = fmaxf(m, pm[a]), b = top == -INFINITY ? 0.f : top;
      const float f0 = ex2_approx(m - b), f1 = ex2_approx(pm[a] - b);
      m = top;
      l = l * f0 + pl[a] * f1;
#pragma unroll
      for (int e = 0; e < COLS; ++e) x[e] = x[e] * f0 + y[a][e] * f1;
    }
  }
  const float inv = l > 0.f ? 1.0f / l : 0.f;
  const int tk = token_of(p, rr);
  uint16_t* dst = p.out + int64_t(s.q0 + tk) * p.o_st + int64_t(cut.h * p.G + rr - tk * p.G) * p.o_sh + col;
#pragma unroll
  for (int e = 0; e < COLS; e += 8)
    *reinterpret_cast<uint4*>(dst + e) = make_uint4(pack_bf16x2(x[e] * inv, x[e + 1] * inv), pack_bf16x2(x[e + 2] * inv, x[e + 3] * inv),
                                                    pack_bf16x2(x[e + 4] * inv, x[e + 5] * inv), pack_bf16x2(x[e + 6] * inv, x[e + 7] * inv));
  if (col == 0) write_lse(p, s, cut.h, rr, m, l);
}

template <int D, int BM, int ROWS>
__global__ void __launch_bounds__(AJ_WARPS * 32) attn_join_kernel(const __grid_constant__ AttnParams p, const Cuts of) {
  griddep_wait();
  join_rows<D, BM, ROWS>(p, of, blockIdx.x + 1, blockIdx.y);
}

template <int D, int COLS, int AHEAD>
__global__ void __launch_bounds__(AJ_WARPS * 32) attn_join_columns_kernel(const __grid_constant__ AttnParams p, const Cuts of) {
  griddep_wait();
  join_columns<D, attn_tc_rows(D), COLS, AHEAD>(p, of, blockIdx.x + 1, blockIdx.y);
}

// Both kernels' units of a mixed batch in one launch.
template <int D, int BM, int ROWS>
__global__ void __launch_bounds__(AJ_WARPS * 32) attn_join_both_kernel(const __grid_constant__ AttnParams p, const Cuts many, const Cuts few) {
  griddep_wait();
  const int of_many = (many.ctas - 1) * many.ys, b = blockIdx.x;
  if (b < of_many)
    join_columns<D, attn_tc_rows(D), D / AJ_WARPS, 1>(p, many, b / many.ys + 1, b % many.ys);
  else
    join_rows<D, BM, ROWS>(p, few, (b - of_many) / few.ys + 1, (b - of_many) % few.ys);
}

// The few-row kernel's cuts and, where there are any, the tcgen05 kernel's.
template <int D, int BM, int ROWS>
cudaError_t join(const AttnParams& p, Cuts few, const Cuts& many, cudaStream_t stream) {
  // rows a unit can have, by the longest sequence the host knows of
  few.ys = (int(std::min<int64_t>(BM, int64_t(p.max_q) * p.G)) + ROWS - 1) / ROWS;
  if (!many.ctas) return launch_behind(attn_join_kernel<D, BM, ROWS>, dim3(few.ctas - 1, few.ys), AJ_WARPS * 32, 0, stream, p, few);
  return launch_behind(attn_join_both_kernel<D, BM, ROWS>, dim3((many.ctas - 1) * many.ys + (few.ctas - 1) * few.ys), AJ_WARPS * 32, 0, stream, p,
                       many, few);
}

template <int D, int WM, int WN, int STAGES, int PER_SM>
cudaError_t run(const AttnParams& p, const AtRows& of, cudaStream_t stream) {
  using C = AtCfg<D, WM, WN, STAGES>;
  static DynSmemCache cache;
  auto kern = attn_kernel<D, WM, WN, STAGES>;
  cudaError_t e = ensure_dyn_smem(reinterpret_cast<const void*>(kern), C::SMEM, cache);
  if (e != cudaSuccess) return e;
  const int ctas = multiprocessor_count() * PER_SM;
  kern<<<ctas, C::THREADS, C::SMEM, stream>>>(p, of);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  return ctas < 2 ? cudaSuccess : join<D, C::BM, C::BM == 16 ? 1 : 2>(p, Cuts{p.ws, of, ctas, 0}, Cuts{}, stream);
}

// `many`: the tcgen05 kernel's cuts, if that has just been launched for the batch's other sequences.  Its parts stay where
// they are, this kernel begins on the multiprocessors that are done with the other, and one join follows (12 sequences
// of 1 to 701 tokens 70 us; one after another, a join each, 73 us).
template <int D, int WM, int WN, int STAGES, int PER_SM>
cudaError_t run_stream(AttnParams p, const AtRows& of, const Cuts& many, cudaStream_t stream) {
  using C = AsCfg<D, WM, WN, STAGES>;
  CUtensorMap maps[2];
  cudaError_t e = encode_kv_maps(p, AT_BN, maps);
  if (e != cudaSuccess) return e;
  static DynSmemCache cache;
  auto kern = attn_stream_kernel<D, WM, WN, STAGES>;
  e = ensure_dyn_smem(reinterpret_cast<const void*>(kern), C::SMEM, cache);
  if (e != cudaSuccess) return e;
  const int ctas = multiprocessor_count() * PER_SM;
  if (many.ctas) {
    p.ws += attn_tc_floats(D);
    e = launch_behind(kern, dim3(ctas), C::THREADS, C::SMEM, stream, p, maps[0], maps[1], of);
  } else {
    kern<<<ctas, C::THREADS, C::SMEM, stream>>>(p, maps[0], maps[1], of);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess || ctas < 2) return e;
  return join<D, C::BM, C::BM == 16 ? 1 : 2>(p, Cuts{p.ws, of, ctas, 0}, many, stream);
}

template <int D, int STAGES, int PER_SM>
cudaError_t pick(const AttnParams& p, int most, const AtRows& of, const Cuts& many, cudaStream_t stream) {
  if (kv_tma_takes(p)) {
    if (most <= 16) return run_stream<D, 1, 4, STAGES, PER_SM>(p, of, many, stream);
    // 32 drafts of 5 tokens over 4000 keys, 32 / 8 heads of 128: 101 us (112 us on tiles of 64 rows)
    if (most <= 32) return run_stream<D, 2, 2, STAGES, PER_SM>(p, of, many, stream);
    return run_stream<D, 4, 1, STAGES, PER_SM>(p, of, many, stream);
  }
  constexpr int S = D == 256 ? 2 : 3;  // pages of any size
  return most <= 16 ? run<D, 1, 4, S, PER_SM>(p, of, stream) : run<D, 4, 1, S, PER_SM>(p, of, stream);
}

cudaError_t small_rows(const AttnParams& p, int most, const AtRows& of, const Cuts& many, cudaStream_t stream) {
  if (p.D == 64) return pick<64, 6, 2>(p, most, of, many, stream);
  if (p.D == 128) return pick<128, 3, 2>(p, most, of, many, stream);
  return pick<256, 3, 1>(p, most, of, many, stream);
}

// Sequences of at most so many rows (tokens times query heads of a key head) are bound by reading their keys
// and stay on warp-level tiles.  Here / on tcgen05, 16 / 2 heads: 64 rows, 32 sequences of 4000 keys, heads of 128 50 / 48 us,
// of 256 81 / 62 us; 32 rows, 8 of 8000 keys, of 128 28 / 34 us, of 256 40 / 42 us; 24 rows, 1 of 20000 keys, of 256 25 / 52 us.
constexpr int few_rows(int head_dim) { return head_dim == 256 ? 32 : 64; }

Cuts tc_cuts(const AttnParams& p, int lo) { return Cuts{p.ws, AtRows{lo, INT32_MAX}, multiprocessor_count(), attn_tc_rows(p.D) / 32}; }

// The tcgen05 kernel's cuts.  A block has all D columns of 32 rows, unless units are few and cut into many parts: then 64
// columns, eight a warp and four parts ahead (40 tokens over 16000 keys, heads of 64 / 128 / 256: 28 / 34 / 36 us a call, not
// 35 / 42 / 42; 2048 tokens over themselves, 2 parts a unit: 36 / 49 / 79 us this way, else 33 / 45 / 75).
template <int D>
cudaError_t tc_join(const AttnParams& p, int lo, cudaStream_t stream) {
  Cuts of = tc_cuts(p, lo);
  if (of.ctas < 2) return cudaSuccess;
  const int64_t units = (int64_t(p.T) * p.G / attn_tc_rows(D) + p.N) * p.Hk;  // or fewer
  if (units * 8 > of.ctas)
    return launch_behind(attn_join_columns_kernel<D, D / AJ_WARPS, 1>, dim3(of.ctas - 1, of.ys), AJ_WARPS * 32, 0, stream, p, of);
  return launch_behind(attn_join_columns_kernel<D, 8, 4>, dim3(of.ctas - 1, of.ys * (D / 64)), AJ_WARPS * 32, 0, stream, p, of);
}

cudaError_t launch_attn_tc_join(const AttnParams& p, int lo, cudaStream_t stream) {
  if (p.D == 64) return tc_join<64>(p, lo, stream);
  if (p.D == 128) return tc_join<128>(p, lo, stream);
  return tc_join<256>(p, lo, stream);
}

}  // namespace

// Strides of one-element dims may be anything: they are not taken.
bool kv_tma_takes(const AttnParams& p) {
  const int64_t strides[6] = {p.k_sh, p.k_st, p.k_sp, p.v_sh, p.v_st, p.v_sp};
  for (int64_t s : strides)
    if (s <= 0 || s % 8 || s * 2 >= (int64_t(1) << 40)) return false;
  return p.page_size % 8 == 0 && p.pages > 0;
}

cudaError_t encode_kv_maps(const AttnParams& p, int bn, CUtensorMap* maps) {
  for (int i = 0; i < 2; ++i) {
    const uint64_t dims[4] = {uint64_t(p.D), uint64_t(p.Hk), uint64_t(p.page_size), uint64_t(p.pages)};
    const uint64_t strides[3] = {uint64_t(i ? p.v_sh : p.k_sh) * 2, uint64_t(i ? p.v_st : p.k_st) * 2, uint64_t(i ? p.v_sp : p.k_sp) * 2};
    const uint32_t box[4] = {64, 1, uint32_t(std::min(p.page_size & -p.page_size, bn)), 1};
    const cudaError_t e = encode_bf16_map(&maps[i], i ? p.v : p.k, 4, dims, strides, box);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

int64_t attn_workspace_bytes(int head_dim) {
  const int64_t ctas = int64_t(multiprocessor_count()) * AT_MAX_CTAS_PER_SM;
  return (attn_tc_floats(head_dim) + ctas * (2 * 64 * (head_dim + 2) + AT_META)) * 4;
}

cudaError_t launch_attn(const AttnParams& p, cudaStream_t stream) {
  const int64_t most = std::min<int64_t>(int64_t(p.max_q) * p.G, INT32_MAX);
  if (most <= few_rows(p.D) || !attn_tc_takes(p)) return small_rows(p, int(most), AtRows{0, INT32_MAX}, Cuts{}, stream);
  const bool alike = int64_t(p.T) == int64_t(p.N) * p.max_q;  // all of the same length
  // sequences of many rows on the tensor-memory tiles, the others, mostly of one token, on tiles of few rows.  The limit is 16
  // rows and not few_rows, although drafts by themselves are better off below that: here the tcgen05 kernel runs anyway, and the
  // other one keeps its smallest tiles.  With 16 / with few_rows, 16 / 2 heads of 64, 128, 256: 32 drafts of 3 to 8 tokens beside a chunk
  // of 2048 over 4096 keys 85 / 92, 103 / 122, 159 / 171 us; 8 of 4 beside 512 over 4096 39 / 47, 49 / 63, 69 / 85 us; 12
  // sequences of 1 to 701 tokens 39 / 43, 49 / 56, 69 / 71 us.
  const int lo = alike ? 0 : (p.G <= 16 ? 16 : few_rows(p.D));
  cudaError_t e = launch_attn_tc(p, lo, stream);
  if (e != cudaSuccess) return e;
  return alike ? launch_attn_tc_join(p, lo, stream) : small_rows(p, lo, AtRows{0, lo}, tc_cuts(p, lo), stream);
}

}  // namespace gdnr
