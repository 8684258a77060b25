/*
 * gdnr.h -- C ABI of the B200-native FP8-checkpoint replay GDN decode path.
 *
 * Every entry point takes plain pointers + shapes + strides (gdnr_tensor),
 * never allocates, never synchronises, and enqueues its work on the CUDA
 * stream it is given (a cudaStream_t passed as void*; NULL = legacy default
 * stream).  Return value: GDNR_OK (0) or a negative gdnr_status; the message
 * of the last failure on the calling thread is gdnr_last_error().
 *
 * Reference interfaces replaced (paths inside zz774ever/fp8-replayssm-gdn-kernel):
 *   gdnr_replay          <- gdn_replay_fp8           prototype/gdn_replayssm_fp8_kernel.py:344-405
 *   gdnr_replay_split    <- gdn_replay_fp8_split     prototype/gdn_replayssm_fp8_kernel.py:1129-1235
 *   gdnr_prep_ring       <- gdn_prep_ring            prototype/gdn_replayssm_fp8_kernel.py:710-795
 *   gdnr_bf16_step       <- gdn_bf16_step            prototype/gdn_replayssm_fp8_kernel.py:408-450
 *   gdnr_quantize_vblock32   <- quantize_checkpoint(state, "vblock", 32)
 *                                                   prototype/gdn_replay_fp8_reference.py:40-106
 *   gdnr_dequantize_vblock32 <- dequantize_checkpoint prototype/gdn_replay_fp8_reference.py:109-134
 *   gdnr_fused_step      <- gdn_prep_ring + gdn_replay_fp8 (+ flush) as one call, the
 *                          full-contract step of prototype/bench_gdn_full_contract.py:138-308
 *
 * Geometry supported by the kernels: K = V = 128 (Qwen3.5 GDN head dims),
 * HV = G*H with G in {1,2,4}, ring length L in [1, 64], one scale per
 * 32 value rows ("vblock32").
 */
#ifndef GDNR_H
#define GDNR_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define GDNR_ABI_VERSION 2 /* 2: adds gdnr_packed_decode (the other structs are unchanged) */

typedef enum {
  GDNR_DT_NONE = 0,
  GDNR_F32 = 1,
  GDNR_F16 = 2,
  GDNR_BF16 = 3,
  GDNR_E4M3 = 4, /* float8_e4m3fn, one byte */
  GDNR_I32 = 5,
  GDNR_U8 = 6,   /* torch.bool / uint8 */
  GDNR_I8 = 7
} gdnr_dtype;

typedef enum {
  GDNR_OK = 0,
  GDNR_ERR_ARG = -1,         /* null pointer, wrong rank, inconsistent shapes */
  GDNR_ERR_DTYPE = -2,       /* unsupported dtype for that argument */
  GDNR_ERR_LAYOUT = -3,      /* stride / 16-byte alignment requirement not met */
  GDNR_ERR_ALIAS = -4,       /* two buffers that must be distinct overlap */
  GDNR_ERR_UNSUPPORTED = -5, /* geometry outside what the kernels implement */
  GDNR_ERR_CUDA = -6         /* launch failed (message has the CUDA error) */
} gdnr_status;

/* Bits of the device error word (see error_flag below). */
#define GDNR_DEVERR_WAIT_TIMEOUT 0x1u /* a bounded mbarrier wait gave up */
#define GDNR_DEVERR_BAD_POS 0x2u      /* fused step: pos[b] outside [0, L); append: positions[t] outside the table */
#define GDNR_DEVERR_BAD_HINT 0x4u     /* flush_hint NONE but a sequence's ring was full; attention: a sequence
                                         longer than max_seqlen */
#define GDNR_DEVERR_BAD_SLOT 0x8u     /* a slot or page outside its pool (packed decode, prompt operators), a
                                         length outside its block table */
#define GDNR_DEVERR_LAYOUT 0x10u      /* a kernel's shared memory did not fit its layout (a launch
                                         configuration fault of the library): nothing was done */

/* flush_hint: what the caller knows about which sequences flush in this call */
#define GDNR_FLUSH_AUTO 0 /* unknown: every head is checked on the device */
#define GDNR_FLUSH_NONE 1 /* no sequence flushes (a full ring is reported as GDNR_DEVERR_BAD_HINT) */
#define GDNR_FLUSH_ALL 2  /* every sequence may flush */

/* launch_flags */
#define GDNR_LAUNCH_PDL 0x1 /* programmatic dependent launch: the kernel may start while the
                               preceding kernel on the stream drains and read this call's
                               checkpoint before that kernel completes.  Only valid when the
                               preceding kernel does not write this call's checkpoint. */

/* Strided view of a device (or, for validation only, any) buffer. */
typedef struct {
  void* data;
  int32_t dtype; /* gdnr_dtype */
  int32_t ndim;  /* 0 = absent (optional argument) */
  int64_t shape[4];
  int64_t stride[4]; /* in elements */
} gdnr_tensor;

/* ---- gdnr_replay: mirror of gdn_replay_fp8 ---------------------------- */
typedef struct {
  gdnr_tensor checkpoint; /* [B,HV,V,K] E4M3, I8 ("vblock_int8" codes, L <= 16; the flush
                             re-quantises to I8), or F32 for the full-precision variant; in/out */
  gdnr_tensor scale;      /* [B,HV,V/32] F16|F32 (absent for an F32 checkpoint); in/out */
  gdnr_tensor q;          /* [B,H,K] BF16|F32, already L2-normalised */
  gdnr_tensor k_ring;     /* [B,L,H,K] BF16 */
  gdnr_tensor v_ring;     /* [B,L,HV,V] BF16 */
  gdnr_tensor g_ring;     /* [B,L,HV] F32|BF16 (log decay) */
  gdnr_tensor beta_ring;  /* [B,L,HV] F32|BF16 */
  gdnr_tensor valid_len;  /* [B] I32: slots 0..valid_len-1 are replayed (clamped to [0,L]) */
  gdnr_tensor flush;      /* [B] U8|I32: nonzero -> rebuild + re-quantise in place */
  gdnr_tensor out;        /* [B,HV,V] BF16|F32 */
  int32_t block_v;        /* value rows per CTA: 32, 64 or 128 (0 -> 128) */
  int32_t quant_divisor;  /* 0: x/(amax/448) like ref.py:94; 1: x/fp16(amax/448) like kern.py:234 */
  uint32_t* error_flag;   /* optional device word, OR-ed with GDNR_DEVERR_* */
  int32_t flush_hint;     /* GDNR_FLUSH_* */
  int32_t launch_flags;   /* GDNR_LAUNCH_* */
} gdnr_replay_args;

int gdnr_replay(const gdnr_replay_args* args, void* stream);

/* ---- gdnr_replay_split: mirror of gdn_replay_fp8_split ----------------- */
typedef struct {
  gdnr_tensor checkpoint, scale, q, k_ring, v_ring, g_ring, beta_ring, valid_len;
  gdnr_tensor tq;   /* [B,HV,K] F32 caller buffer: receives the transformed query */
  gdnr_tensor coef; /* [B,HV,L] F32 caller buffer: receives c_t for t < valid_len */
  gdnr_tensor out;  /* [B,HV,V] BF16|F32 */
  int32_t block_v;
  uint32_t* error_flag;
} gdnr_replay_split_args;

int gdnr_replay_split(const gdnr_replay_split_args* args, void* stream);

/* ---- gdnr_replay_split_static: gdnr_replay_split without caller scratch --
 * No counterpart in the reference.  The split replay needs T [B,HV,K] and
 * c [B,HV,L] scratch; this entry point keeps them in a library-owned device
 * array instead, for callers that cannot allocate device memory when they
 * call the replay (e.g. a serving runtime that reserves all device memory for
 * its state pool up front, or code inside an allocator callback that must not
 * re-enter the allocator).  It allocates nothing.
 *
 * Limits: B*HV <= GDNR_SPLIT_STATIC_MAX_PAIRS and L <= GDNR_SPLIT_STATIC_MAX_L
 * (3 MiB of scratch per device); larger calls fail with GDNR_ERR_UNSUPPORTED.
 * The first call on a device looks up the scratch address (cudaGetSymbolAddress,
 * with that device current) and caches it: make that first call before any
 * stream capture.  All calls on a device share the one scratch, so calls that
 * overlap in time (concurrent streams or host threads) race on it; serialise
 * them.  Nothing in the scratch needs to start at zero. */
#define GDNR_SPLIT_STATIC_MAX_PAIRS 4096
#define GDNR_SPLIT_STATIC_MAX_L 64
typedef struct {
  gdnr_tensor checkpoint, scale, q, k_ring, v_ring, g_ring, beta_ring, valid_len; /* as gdnr_replay_split */
  gdnr_tensor out;
  int32_t block_v;
  uint32_t* error_flag;
} gdnr_replay_split_static_args;

int gdnr_replay_split_static(const gdnr_replay_split_static_args* args, void* stream);

/* ---- gdnr_prep_ring: mirror of gdn_prep_ring --------------------------- */
typedef struct {
  gdnr_tensor mixed_qkv; /* [B, 2*H*K + HV*V] BF16|F32, inner stride 1 */
  gdnr_tensor a, b;      /* [B,HV] BF16|F32 */
  gdnr_tensor a_log;     /* [HV] F32 */
  gdnr_tensor dt_bias;   /* [HV] F32 */
  gdnr_tensor pos;       /* [B] I32 ring slot written */
  gdnr_tensor q_out;     /* [B,H,K] BF16|F32 */
  gdnr_tensor k_ring, v_ring, g_ring, beta_ring;
  uint32_t* error_flag;
} gdnr_prep_args;

int gdnr_prep_ring(const gdnr_prep_args* args, void* stream);

/* ---- gdnr_fused_step: prep + ring append + replay + flush, one launch -- */
typedef struct {
  gdnr_tensor mixed_qkv, a, b, a_log, dt_bias; /* as gdnr_prep_args */
  gdnr_tensor pos;        /* [B] I32: slot of this token; the step flushes when pos == L-1 */
  gdnr_tensor pos_out;    /* optional [B] I32 (distinct from pos): receives (pos+1) % L */
  gdnr_tensor checkpoint; /* [B,HV,V,K] E4M3 | I8 (L <= 16) | F32, in/out */
  gdnr_tensor scale;      /* [B,HV,V/32] F16|F32 (absent for F32 checkpoint), in/out */
  gdnr_tensor k_ring, v_ring, g_ring, beta_ring; /* in/out: slot pos is written */
  gdnr_tensor out;        /* [B,HV,V] BF16|F32 */
  gdnr_tensor q_out;      /* optional [B,H,K]: normalised q as the reference's prep writes it */
  int32_t quant_divisor;
  uint32_t* error_flag;
  int32_t flush_hint;     /* GDNR_FLUSH_* */
  int32_t launch_flags;   /* GDNR_LAUNCH_* */
} gdnr_step_args;

int gdnr_fused_step(const gdnr_step_args* args, void* stream);

/* ---- gdnr_packed_decode: the production decode call over a state-slot pool --
 * Replaces the serving engine's decode call
 *   fused_recurrent_gated_delta_rule_packed_decode(mixed_qkv, a, b, A_log, dt_bias, scale,
 *       initial_state, out, ssm_state_indices, use_qk_l2norm_in_kernel=True)
 * as the reference drives it (prototype/bench_gdn_full_contract.py:157-170; contract notes
 * findings.md:37-45), with the bf16 state cache [slots,HV,V,K] replaced by the FP8
 * checkpoint + ring pool below: batch row i uses slot state_indices[i] of every state
 * tensor.  An index <= 0 is the null slot (the serving engine's padding; the production
 * kernel's NULL_BLOCK_ID test, vLLM fused_recurrent.py:292-297): no state is read or written
 * for that row and its out rows are written as zeros, as the production op does.  An index
 * >= slots is treated the same way and reported as GDNR_DEVERR_BAD_SLOT.  The non-null
 * indices of one call must be distinct (one row per sequence, as in the production
 * contract): two rows on one slot race on its state within the launch and the result is
 * undefined; nothing checks for it.  q and k are
 * always L2-normalised in the kernel and the output is scaled by K^-1/2: the production
 * call's use_qk_l2norm_in_kernel and scale arguments must be 1 and K^-1/2.  The step is
 * gdnr_fused_step's (prep + ring append + replay, and the flush when a slot's pos is L-1);
 * pos_out (optional, [slots]) receives (pos+1) % L for the slots of the batch.  E4M3
 * checkpoints only, in the layout gdnr_fused_step's persistent kernel takes (16-byte
 * aligned rows and rings, HV/H = 1 or even, 4 <= L <= 16); anything else fails with
 * GDNR_ERR_UNSUPPORTED. */
typedef struct {
  gdnr_tensor mixed_qkv, a, b, a_log, dt_bias; /* [B,...] as gdnr_step_args */
  gdnr_tensor state_indices; /* [B] I32: slot of each batch row */
  gdnr_tensor pos;        /* [slots] I32: ring slot of this token, per state slot */
  gdnr_tensor pos_out;    /* optional [slots] I32 (distinct from pos) */
  gdnr_tensor checkpoint; /* [slots,HV,V,K] E4M3, in/out */
  gdnr_tensor scale;      /* [slots,HV,V/32] F16|F32, in/out */
  gdnr_tensor k_ring, v_ring, g_ring, beta_ring; /* [slots,L,...] in/out */
  gdnr_tensor out;        /* [B,HV,V] or [B,1,HV,V] BF16|F32 */
  float qk_scale;         /* must be K^-1/2 */
  int32_t use_qk_l2norm;  /* must be 1 */
  int32_t quant_divisor;
  uint32_t* error_flag;
  int32_t flush_hint;     /* GDNR_FLUSH_* */
  int32_t launch_flags;   /* GDNR_LAUNCH_*; GDNR_LAUNCH_PDL is accepted, but the early
                             checkpoint requests wait for griddepcontrol.wait here (the
                             slots come from state_indices, an input) */
} gdnr_packed_decode_args;

int gdnr_packed_decode(const gdnr_packed_decode_args* args, void* stream);

/* ---- FP8 vblock32 codec ------------------------------------------------ */
typedef struct {
  gdnr_tensor state;      /* [B,HV,V,K] F32 (quantize: in; dequantize: out) */
  gdnr_tensor payload;    /* [B,HV,V,K] E4M3 */
  gdnr_tensor scale;      /* [B,HV,V/32] F16|F32 */
  int32_t quant_divisor;  /* as gdnr_replay_args */
  uint32_t* saturation_count; /* optional device counter: += #{|x/divisor| > 448} */
} gdnr_codec_args;

int gdnr_quantize_vblock32(const gdnr_codec_args* args, void* stream);
int gdnr_dequantize_vblock32(const gdnr_codec_args* args, void* stream);

/* ---- gdnr_bf16_step: mirror of gdn_bf16_step (bf16 state RMW control) -- */
typedef struct {
  gdnr_tensor state; /* [B,HV,V,K] BF16, in/out */
  gdnr_tensor q, k;  /* [B,H,K] BF16|F32 */
  gdnr_tensor v;     /* [B,HV,V] BF16|F32 */
  gdnr_tensor g, beta; /* [B,HV] BF16|F32 */
  gdnr_tensor out;   /* [B,HV,V] BF16|F32 */
} gdnr_bf16_step_args;

int gdnr_bf16_step(const gdnr_bf16_step_args* args, void* stream);

/* ==== prompts and mixed batches of a hybrid model =========================
 * No counterparts in the reference: what a process that serves a hybrid model
 * (GDN layers and softmax-attention layers) calls next to the decode step above.
 *
 * A ragged batch of N sequences is packed: the tokens of sequence n are rows
 * cu_seqlens[n] .. cu_seqlens[n+1]-1 of the token tensors (cu_seqlens [N+1] I32,
 * ascending from 0; a sequence may be empty).  max_seqlen is the longest of them as far
 * as the host knows it (0: unknown); it picks kernels and grids.  gdnr_paged_attention
 * reports a longer one as GDNR_DEVERR_BAD_HINT, and its rows may be incomplete.  Token
 * rows that belong to no sequence are not written. */

/* ---- gdnr_gdn_prefill: the gated delta rule over whole sequences ----------
 * Per value head, token by token, with k = k_raw / sqrt(|k_raw|^2 + 1e-6), q likewise
 * times K^-1/2, g = -exp(A_log) softplus(a + dt_bias), beta = sigmoid(b):
 *   S <- e^g S;  S <- S + beta (v - S k) k^T;  out = S q
 * The state is float32 throughout; normalised keys are not rounded (the decode step's
 * ring holds them in bf16).  state_indices as in gdnr_packed_decode: sequence n uses
 * slot state_indices[n]; an index <= 0 is the null slot (out rows are zeros, no state is
 * touched), one >= slots likewise and reported as GDNR_DEVERR_BAD_SLOT; the non-null ones
 * must be distinct.  Without it sequence n uses slot n.  has_initial[n] == 0: the
 * sequence starts from the zero state and its slot is only written.
 *
 * All sequences of a call go one way, token by token or in chunks of 64 tokens; max_seqlen
 * decides (more than 20: chunks), or the mean length where it is 0.  In chunks, single tokens
 * beside a long prompt cost a chunk each: give them a call of their own where they are many.
 * A value that is not finite spoils its sequence's rows from its chunk on, earlier tokens of that
 * chunk among them. */
typedef struct {
  gdnr_tensor mixed_qkv;     /* [T, 2*H*K + HV*V] BF16, raw q | k | v */
  gdnr_tensor a, b;          /* [T,HV] BF16|F16|F32 */
  gdnr_tensor a_log;         /* [HV] F32 */
  gdnr_tensor dt_bias;       /* [HV] F32 */
  gdnr_tensor state;         /* [slots,HV,V,K] F32, in/out */
  gdnr_tensor cu_seqlens;    /* [N+1] I32, contiguous */
  gdnr_tensor state_indices; /* optional [N] I32 */
  gdnr_tensor has_initial;   /* optional [N] U8 (absent: every sequence continues its slot) */
  gdnr_tensor out;           /* [T,HV,V] BF16 */
  int32_t max_seqlen;
  int32_t reserved;
  void* workspace;           /* gdnr_gdn_prefill_workspace() bytes (may be 0), 16-byte aligned,
                                private to the call until it has run; need not be zero */
  int64_t workspace_bytes;
  uint32_t* error_flag;
} gdnr_prefill_args;

int gdnr_gdn_prefill(const gdnr_prefill_args* args, void* stream);
/* Workspace bytes of gdnr_gdn_prefill for T tokens of N sequences: in chunks 21568 bytes for each of
 * (T / 64 + N) chunks of each value head (at 32 heads 11 KB a token and 690 KB a sequence), none token
 * by token. */
int64_t gdnr_gdn_prefill_workspace(int64_t tokens, int64_t sequences, int32_t value_heads, int32_t max_seqlen);

/* ---- gdnr_qk_norm_rope_append --------------------------------------------
 * Per token and head: x / sqrt(mean(x^2) + eps) * (weight + weight_offset) for queries
 * and keys (each only with its weight), the rotation of the first `rot` elements by row
 * positions[t] of cos_sin (cos of the rot/2 angles, then sin), pairs (i, i + rot/2) or,
 * interleaved, (2i, 2i + 1); then q to q_out, k and v to slot slots[t] (page slots[t] /
 * page_size, row slots[t] % page_size) of the caches.  slots[t] < 0: padding, nothing
 * is appended.  A slot past the cache sets GDNR_DEVERR_BAD_SLOT and is not
 * written; a position outside the table sets GDNR_DEVERR_BAD_POS and leaves q and k
 * unrotated.  Head dim D = 64, 128 or 256. */
typedef struct {
  gdnr_tensor q;         /* [T,Hq,D] BF16 (rows 16-byte aligned, as all below) */
  gdnr_tensor k, v;      /* [T,Hk,D] BF16 */
  gdnr_tensor q_weight, k_weight; /* optional [D] BF16|F32, contiguous, 16-byte aligned */
  gdnr_tensor positions; /* [T] I32 */
  gdnr_tensor slots;     /* [T] I32, distinct where >= 0 */
  gdnr_tensor cos_sin;   /* [P, rot] F32 */
  gdnr_tensor q_out;     /* [T,Hq,D] BF16 (may be q itself) */
  gdnr_tensor k_cache, v_cache; /* [pages,page_size,Hk,D] BF16, in/out */
  float eps;
  float weight_offset;
  int32_t interleaved;
  int32_t reserved;
  uint32_t* error_flag;
} gdnr_append_args;

int gdnr_qk_norm_rope_append(const gdnr_append_args* args, void* stream);

/* ---- gdnr_paged_attention --------------------------------------------------
 * The m new tokens of a sequence (its rows of q) are the last m of its kv_lens[n]
 * cached ones: row i attends places 0 .. kv_lens[n] - m + i (causal).  A row that
 * sees no place is zero with lse -inf.  Query head h reads key head h / (Hq/Hk).
 * What pages hold past a sequence's end is never used; the values of the places
 * before it are expected to be finite.  block_table[n][j] is the page of places
 * j*page_size ..; entries beyond the sequence's pages are not read.  A page outside the
 * cache sets GDNR_DEVERR_BAD_SLOT and reads as zeros.  So does a kv_lens[n] below zero or past
 * the block table (width*page_size places) where the sequence has rows: they are
 * computed as if it were zero, or the table's places. */
typedef struct {
  gdnr_tensor q;           /* [T,Hq,D] BF16, D = 64, 128 or 256 */
  gdnr_tensor k_cache, v_cache; /* [pages,page_size,Hk,D] BF16 */
  gdnr_tensor block_table; /* [N,width] I32 */
  gdnr_tensor kv_lens;     /* [N] I32 */
  gdnr_tensor cu_seqlens;  /* [N+1] I32, contiguous */
  gdnr_tensor out;         /* [T,Hq,D] BF16 */
  gdnr_tensor lse;         /* optional [T,Hq] F32: log of the row's sum of exp(score) */
  float scale;
  int32_t max_seqlen;
  void* workspace;         /* gdnr_paged_attention_workspace(D) bytes, 16-byte aligned, private
                              to the call until it has run; need not be zero */
  int64_t workspace_bytes;
  uint32_t* error_flag;
} gdnr_attn_args;

int gdnr_paged_attention(const gdnr_attn_args* args, void* stream);
/* Workspace bytes of gdnr_paged_attention on the current device for head dim D, whatever the batch: every
 * multiprocessor's parts of units that are cut (148 of them: 30, 59 and 78 MB for D = 64, 128 and 256). */
int64_t gdnr_paged_attention_workspace(int32_t head_dim);

/* ---- misc --------------------------------------------------------------- */
const char* gdnr_last_error(void);
const char* gdnr_version(void);
int gdnr_abi_version(void);
/* Library-owned device error word used when a call passes error_flag = NULL.
 * Reads it (synchronously, on the current device) and optionally clears it. */
int gdnr_read_device_error(uint32_t* value, int clear);

/* Diagnostic, no counterpart in the reference: one tiny launch that runs the
 * persistent step kernel's bounded-wait code into its time limit (a barrier
 * nothing arrives on, held with 32 tensor-memory columns allocated) and
 * returns cleanly.  After it completes (about one second of GPU time), the
 * error word has GDNR_DEVERR_WAIT_TIMEOUT set and report (device memory,
 * 4 x u64) holds: both waits' results (0 = gave up), then the nanoseconds
 * each waited; the second wait ends through the abort word the first one set.
 * Used by the tests to show that a timed-out wait leaves the context usable. */
int gdnr_selftest_wait_timeout(uint32_t* error_flag, unsigned long long* report, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* GDNR_H */
