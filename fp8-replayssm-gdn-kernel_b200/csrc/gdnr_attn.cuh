// Work split of the paged-attention kernels: units, equal shares, and how a cut unit is joined.
#pragma once

#include "gdnr_device.cuh"
#include "gdnr_hybrid.h"
#include "gdnr_tile.cuh"

namespace gdnr {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr int AT_META = 8;  // ints of one CTA's record

// A kernel's tiles: BM rows (token, query head) by BN keys, for the sequences whose rows are in (lo, hi].
// OVER: what beginning and ending a unit costs, in tiles.
template <int BM_, int BN_, int OVER_>
struct AtTile {
  static constexpr int BM = BM_, BN = BN_, OVER = OVER_;
};

struct AtRows {
  int lo, hi;
};

struct SeqLen {
  int q0, m, kv;
};

__device__ __forceinline__ SeqLen seq_len(const AttnParams& p, int n) {
  SeqLen s;
  s.q0 = min(max(p.cu[n], 0), p.T);
  s.m = min(max(p.cu[n + 1], s.q0), p.T) - s.q0;
  s.kv = int(min(int64_t(max(p.kv_lens[n * p.kl_s], 0)), int64_t(p.width) * p.page_size));
  return s;
}

// As seq_len, without rows where the sequence is another kernel's.
__device__ __forceinline__ SeqLen seq_len(const AttnParams& p, int n, const AtRows& r) {
  SeqLen s = seq_len(p, n);
  if (s.m * p.G <= r.lo || s.m * p.G > r.hi) s.m = 0;
  return s;
}

// row / G: a multiplication where that is exact for every row (the host checks)
__device__ __forceinline__ int token_of(const AttnParams& p, int row) {
  return p.g_magic ? int(__umulhi(uint32_t(row), p.g_magic)) : row / p.G;
}

// Keys that rows up to (not including) `rows` of a sequence see.
__device__ __forceinline__ int keys_seen(const AttnParams& p, const SeqLen& s, int rows) {
  return min(s.kv, s.kv - s.m + token_of(p, min(rows, s.m * p.G) - 1) + 1);
}

// A unit is (sequence, key head, tile of BM rows); its cost is the number of key tiles
// its last row sees, and OVER places before them.  The units of the batch laid end to end are cut into
// equal shares, one per CTA, so ragged lengths and few heads fill the machine alike.  A cut among a unit's
// first OVER places leaves the unit whole, to the later share.
template <class T>
__device__ __forceinline__ int unit_tiles(const AttnParams& p, const SeqLen& s, int rt) {
  return max(1, (keys_seen(p, s, (rt + 1) * T::BM) + T::BN - 1) / T::BN);  // a unit without keys still writes its rows
}

// A warp looks at 32 / per sequences at a time with `per` lanes each, so that one long sequence does not
// keep a single lane busy.
__device__ __forceinline__ int lanes_per_seq(int n) { return n >= 32 ? 1 : (n > 16 ? 1 : (n > 8 ? 2 : (n > 4 ? 4 : (n > 2 ? 8 : (n > 1 ? 16 : 32))))); }

// Places of one head of sequence n (0 past the last), in each of its `per` lanes.
template <class T>
__device__ __forceinline__ int64_t seq_tiles(const AttnParams& p, const AtRows& r, int n, int per, int lane) {
  int64_t sum = 0;
  if (n < p.N) {
    const SeqLen s = seq_len(p, n, r);
    const int rts = (s.m * p.G + T::BM - 1) / T::BM;
    for (int rt = lane & (per - 1); rt < rts; rt += per) sum += T::OVER + unit_tiles<T>(p, s, rt);
  }
  for (int o = per >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}

// The warps of a CTA count the batch's places together: warp w the sequences [w per, (w + 1) per), all of a short batch
// by the first.
__device__ __forceinline__ int seqs_per_warp(const AttnParams& p, int warps) { return p.N <= 32 ? p.N : (p.N + warps - 1) / warps; }

// Places of a warp's sequences.
template <class T>
__device__ __forceinline__ int64_t warp_places(const AttnParams& p, const AtRows& r, int warp, int warps, int lane) {
  const int first = warp * seqs_per_warp(p, warps), last = min(first + seqs_per_warp(p, warps), p.N);
  const int per = lanes_per_seq(last - first), step = 32 / per;
  int64_t w = 0;
  for (int n0 = first; n0 < last; n0 += step) {
    const int n = n0 + lane / per;
    const int64_t x = seq_tiles<T>(p, r, n < last ? n : p.N, per, lane);
    if ((lane & (per - 1)) == 0) w += x * p.Hk;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
  return w;
}

struct Unit {
  int n, h, rt;
  SeqLen s;
  int64_t begin;  // first place of the unit
  int tiles;
};

// The unit that place `at` of the batch falls into (one whole warp); places: every warp's, as warp_places counts them.
template <class T>
__device__ __forceinline__ Unit find_unit(const AttnParams& p, const AtRows& r, int64_t at, const int64_t* places, int warps, int lane) {
  int64_t base = 0;
  int first = 0;
  const int mine = seqs_per_warp(p, warps);
  for (int w = 0; w + 1 < warps && base + places[w] <= at; ++w) base += places[w], first += mine;
  const int last = min(first + mine, p.N), per = lanes_per_seq(last - first), step = 32 / per;
  Unit u;
  u.n = 0, u.h = 0, u.rt = 0, u.begin = 0, u.tiles = 0;
  u.s.q0 = u.s.m = u.s.kv = 0;
  for (int n0 = first; n0 < last; n0 += step) {
    const int n = n0 + lane / per;
    const int64_t head = seq_tiles<T>(p, r, n < last ? n : p.N, per, lane), w = head * p.Hk;
    int64_t pre = w;
    for (int o = per; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, pre, o);
      if (lane >= o) pre += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, base + pre > at);
    if (hit) {
      const int src = __ffs(hit) - 1;
      int64_t start = base + __shfl_sync(0xffffffffu, pre - w, src);
      u.n = n0 + src / per;
      u.s = seq_len(p, u.n, r);
      const int64_t per_head = __shfl_sync(0xffffffffu, head, src);
      u.h = at - start < INT32_MAX ? int(uint32_t(at - start) / uint32_t(min(per_head, int64_t(INT32_MAX)))) : int((at - start) / per_head);
      start += u.h * per_head;
      const int rts = (u.s.m * p.G + T::BM - 1) / T::BM;
      if (rts == 1) {
        u.tiles = int(per_head) - T::OVER;
        u.begin = start;
        return u;
      }
      for (int rt0 = 0; rt0 < rts; rt0 += 32) {
        const int own = rt0 + lane < rts ? T::OVER + unit_tiles<T>(p, u.s, rt0 + lane) : 0;
        int sum = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += v;
        }
        const unsigned in = __ballot_sync(0xffffffffu, start + sum > at);
        if (in) {
          const int l = __ffs(in) - 1;
          u.rt = rt0 + l;
          u.tiles = __shfl_sync(0xffffffffu, own, l) - T::OVER;
          u.begin = start + __shfl_sync(0xffffffffu, sum - own, l);
          return u;
        }
        start += __shfl_sync(0xffffffffu, sum, 31);
      }
    }
    base += __shfl_sync(0xffffffffu, pre, 31);
  }
  u.n = p.N;
  return u;
}

// The next unit in order.
template <class T>
__device__ __forceinline__ void next_unit(const AttnParams& p, const AtRows& r, Unit& u) {
  u.begin += T::OVER + u.tiles;
  ++u.rt;
  if (u.rt * T::BM >= u.s.m * p.G) {
    u.rt = 0;
    if (++u.h == p.Hk) {
      u.h = 0;
      do {
        if (++u.n >= p.N) return;
        u.s = seq_len(p, u.n, r);
      } while (u.s.m == 0);
    }
  }
  u.tiles = unit_tiles<T>(p, u.s, u.rt);
}

struct Share {
  int64_t begin, end;
};

// Shares of `total` places: no more than units of one tile would give, so that small batches do not pay for joining.
template <class T>
__device__ __forceinline__ int64_t shares(int64_t total, int ctas) {
  return min(int64_t(ctas), (total + T::OVER) / (T::OVER + 1));
}

// Share i: sizes differ by one at most, the larger ones first.
template <class T>
__device__ __forceinline__ Share share_of(int64_t total, int i, int ctas) {
  const int64_t use = shares<T>(total, ctas);
  Share s;
  if (i >= use) {
    s.begin = s.end = total;
    return s;
  }
  const int64_t size = total < INT32_MAX ? int32_t(total) / int32_t(use) : total / use, more = total - size * use;
  s.begin = size * i + min(int64_t(i), more);
  s.end = s.begin + size + (i < more ? 1 : 0);
  return s;
}

// The share that place `at` falls into.
template <class T>
__device__ __forceinline__ int share_at(int64_t total, int64_t at, int ctas) {
  const int64_t use = shares<T>(total, ctas), size = total / use, more = total - size * use;
  return int(at < more * (size + 1) ? at / (size + 1) : more + (at - more * (size + 1)) / size);
}

// Key tiles of the unit that a share has.
struct Tiles {
  int begin, end;
};

template <class T>
__device__ __forceinline__ Tiles tiles_of(const Share& s, const Unit& u) {
  Tiles t;
  t.begin = int(max(s.begin - u.begin - T::OVER, int64_t(0)));
  t.end = int(max(min(s.end - u.begin - T::OVER, int64_t(u.tiles)), int64_t(0)));
  return t;
}

// A CTA's record for the join, in the workspace behind the parts [ctas][2][BM][D + 2]: a share that
// begins inside a unit leaves its part of it in slot 0, one that only ends inside in slot 1.
template <class T>
__device__ __forceinline__ void write_meta(int* meta, const Share& share, const Unit& u, int64_t total, int ctas) {
  const int64_t before = share.begin - u.begin - T::OVER;  // tiles of the unit in earlier shares
  int4* const to = reinterpret_cast<int4*>(meta);
  // the unit this share continues (n = -1: none) and the share of its last tile
  to[0] = make_int4(before > 0 ? u.n : -1, u.h, u.rt, int(max(before, int64_t(0))));
  to[1] = make_int4(share_at<T>(total, u.begin + T::OVER + u.tiles - 1, ctas), int(share.end - share.begin), 0, 0);
}

// What a join's block reads of share i: false where no unit is cut between shares i - 1 and i, or not for the
// first time.
struct CutUnit {
  int n, h, rt, parts;  // parts: shares i - 1 .. the one of the unit's last tile
};

__device__ __forceinline__ bool cut_unit(const int* metas, int i, CutUnit& c) {
  const int4 a = *reinterpret_cast<const int4*>(metas + i * AT_META), b = *reinterpret_cast<const int4*>(metas + i * AT_META + 4);
  const int before = metas[(i - 1) * AT_META + 5];  // places of the share before
  c.n = a.x, c.h = a.y, c.rt = a.z, c.parts = b.x - i + 2;
  return a.x >= 0 && before >= a.w;  // else share i - 1 continues the unit, too
}

// What a unit's sequence has that is not in order (one thread).  Only a length that is zero or fills the block table may have
// been cut by seq_len: only then is it read again.
__device__ __forceinline__ void report_unit(const AttnParams& p, const Unit& u) {
  const int64_t most = int64_t(p.width) * p.page_size;
  if (u.s.m > p.max_q) atomicOr(p.err, GDNR_DEVERR_BAD_HINT);  // the join's grid goes by max_q
  if (u.s.kv == 0 || u.s.kv == most) {
    const int kv = p.kv_lens[u.n * p.kl_s];
    if (kv < 0 || kv > most) atomicOr(p.err, GDNR_DEVERR_BAD_SLOT);
  }
}

// Row r of a sequence: token q0 + r / G, query head h G + r % G.
__device__ __forceinline__ int64_t out_at(const AttnParams& p, const Unit& u, int row) {
  const int t = token_of(p, row);
  return int64_t(u.s.q0 + t) * p.o_st + int64_t(u.h * p.G + row - t * p.G) * p.o_sh;
}

// -inf marks a row that saw no place (a sum of zero); a sum of NaN, from a NaN in the row or in a key it saw, stays one.
__device__ __forceinline__ void write_lse(const AttnParams& p, const SeqLen& s, int h, int row, float max2, float sum) {
  if (!p.lse) return;
  const int t = token_of(p, row);
  p.lse[int64_t(s.q0 + t) * p.l_st + int64_t(h * p.G + row - t * p.G) * p.l_sh] = sum == 0.f ? -INFINITY : (max2 + log2f(sum)) * LN2;
}

// ---------------------------------------------------------------- keys and values by TMA
// Tiles of BN keys as boxes of 64 elements by gcd(page_size, BN) rows of one page: whole 8-row swizzle patterns
// where the page size is a multiple of 8.
bool kv_tma_takes(const AttnParams& p);
cudaError_t encode_kv_maps(const AttnParams& p, int bn, CUtensorMap* maps);

__device__ __forceinline__ void kv_tma(uint32_t dst, const CUtensorMap* map, int c, int h, int off, int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(c), "r"(h), "r"(off), "r"(page), "r"(smem_addr(bar))
      : "memory");
}

// The box of tile t that a lane requests: a page past the sequence's end, or outside the cache, reads as zeros
// (its coordinate lies past the map).
struct KvBox {
  bool live;
  int col, off, page;
  uint32_t to;  // byte offset in the tile [ATOMS][BN][128 bytes]
};

template <int BN, int ATOMS>
__device__ __forceinline__ KvBox kv_box(const AttnParams& p, const Unit& u, const int32_t* table, int t, int lane) {
  const int rows = min(p.page_size & -p.page_size, BN), atom = lane % ATOMS, part = lane / ATOMS, tok = t * BN + part * rows;
  KvBox b;
  b.live = part * rows < BN;
  b.col = atom * 64;
  b.to = atom * (BN * 128) + part * rows * 128;
  b.page = p.pages, b.off = 0;
  if (b.live && tok < u.s.kv) {
    const int pi = p.page_shift >= 0 ? tok >> p.page_shift : tok / p.page_size;
    b.page = table[pi];
    b.off = tok - pi * p.page_size;
    if (b.page < 0 || b.page >= p.pages) {
      b.page = p.pages, b.off = 0;
      atomicOr(p.err, GDNR_DEVERR_BAD_SLOT);
    }
  }
  return b;
}

// Tiles on the fifth-generation tensor cores (gdnr_attn_tc.cu): sequences of more than `lo` rows, in tiles of attn_tc_rows.
// Its parts and records are the first attn_tc_floats of the workspace; the join (gdnr_attn.cu) has to follow.
constexpr int attn_tc_rows(int head_dim) { return head_dim == 256 ? 128 : 256; }
bool attn_tc_takes(const AttnParams& p);
int64_t attn_tc_floats(int head_dim);
cudaError_t launch_attn_tc(const AttnParams& p, int lo, cudaStream_t stream);

}  // namespace gdnr
