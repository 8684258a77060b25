// Parameter blocks and launchers of the prompt / mixed-batch operators of a
// hybrid model: gated delta rule over ragged sequences (gdnr_prefill.cu), norm +
// rotation + cache append (gdnr_append.cu), attention over a paged cache
// (gdnr_attn.cu).  Strides are in elements.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "gdnr_internal.h"

namespace gdnr {

struct PrefillParams {
  const uint16_t* mixed;  // [T, 2HK + HV V] bf16
  int64_t mx_s;
  const void* a;
  int64_t a_st, a_sh;
  int32_t a_dt;
  const void* b;
  int64_t b_st, b_sh;
  int32_t b_dt;
  const float* a_log;
  int64_t al_s;
  const float* dt_bias;
  int64_t db_s;
  float* state;  // [S, HV, 128, 128], rows packed
  int64_t st_ss, st_sh;
  const int32_t* cu;  // [N+1]
  const int32_t* sidx;  // optional [N]
  int64_t si_s;
  const uint8_t* has_init;  // optional [N]
  int64_t hi_s;
  uint16_t* out;  // [T, HV, V] bf16
  int64_t o_st, o_sh;
  int32_t N, H, HV, S, T;
  uint8_t* images;  // chunked form: workspace, CK_IMAGE_BYTES a chunk and value head
  bool whole;       // set by the launcher: the images hold T whole
  uint32_t* err;
};

constexpr int CK_IMAGE_BYTES = 21568;

// Tokens [begin, end) of sequence n and the slot of its state; returns false for a
// null or out-of-range slot (rows become zeros, no state is touched).
struct SeqRange {
  int begin, end, slot;
};

__device__ __forceinline__ SeqRange prefill_seq(const PrefillParams& p, int n) {
  SeqRange r;
  // clamped, so that offsets that do not ascend within [0, T] cannot reach outside the tensors
  r.begin = min(max(p.cu[n], 0), p.T);
  r.end = min(max(p.cu[n + 1], r.begin), p.T);
  r.slot = n;
  if (p.sidx) {
    r.slot = p.sidx[n * p.si_s];
    if (r.slot >= p.S) {
      atomicOr(p.err, GDNR_DEVERR_BAD_SLOT);
      r.slot = 0;
    }
    if (r.slot <= 0) r.slot = -1;
  }
  return r;
}

cudaError_t launch_prefill_recurrent(const PrefillParams& p, cudaStream_t stream);
cudaError_t launch_prefill_chunk(PrefillParams p, int64_t longest, cudaStream_t stream);
// max_seqlen: 0 where the host does not know it
int64_t prefill_workspace_bytes(int64_t tokens, int64_t sequences, int64_t value_heads, int max_seqlen);
cudaError_t launch_prefill(const PrefillParams& p, int max_seqlen, cudaStream_t stream);

struct AppendParams {
  const uint16_t *q, *k, *v;  // [T, Hq|Hk, D] bf16
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
  const void *qw, *kw;  // optional [D]
  int32_t qw_dt, kw_dt;
  const int32_t* pos;
  int64_t pos_s;
  const int32_t* slots;
  int64_t sl_s;
  const float* table;  // [P, rot]: cos | sin
  int64_t tb_s;
  uint16_t* q_out;  // [T, Hq, D]
  int64_t qo_st, qo_sh;
  uint16_t *kc, *vc;  // [pages, page_size, Hk, D]
  int64_t kc_sp, kc_st, kc_sh, vc_sp, vc_st, vc_sh;
  int32_t T, Hq, Hk, D, rot, P, pages, page_size, page_shift, inter, tb_vec;
  float eps, w_off;
  uint32_t* err;
};

cudaError_t launch_append(const AppendParams& p, cudaStream_t stream);

struct AttnParams {
  const uint16_t* q;  // [T, Hq, D]
  int64_t q_st, q_sh;
  const uint16_t *k, *v;  // [pages, page_size, Hk, D]
  int64_t k_sp, k_st, k_sh, v_sp, v_st, v_sh;
  const int32_t* table;  // [N, width]
  int64_t tb_s;
  const int32_t* kv_lens;
  int64_t kl_s;
  const int32_t* cu;
  uint16_t* out;  // [T, Hq, D]
  int64_t o_st, o_sh;
  float* lse;  // optional [T, Hq]
  int64_t l_st, l_sh;
  float scale;
  int32_t N, T, Hq, Hk, G, D, pages, page_size, page_shift, width, max_q;
  uint32_t g_magic;  // row / G = high half of row * g_magic; 0: divide
  float* ws;
  int64_t ws_bytes;
  uint32_t* err;
};

int64_t attn_workspace_bytes(int head_dim);
cudaError_t launch_attn(const AttnParams& p, cudaStream_t stream);

int multiprocessor_count();

// Tiled map of a bf16 tensor, 128-byte swizzle (boxes of 64 innermost elements); strides in bytes, without the innermost.
cudaError_t encode_bf16_map(CUtensorMap* map, const void* base, int rank, const uint64_t* dims, const uint64_t* strides,
                            const uint32_t* box);

// Launches a kernel that may be set up while the one before it in the stream still runs; it waits for that one's
// results itself (griddep_wait).
template <class K, class... A>
cudaError_t launch_behind(K kern, dim3 grid, int threads, int smem, cudaStream_t stream, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

}  // namespace gdnr
