// extern "C" entry points of the prompt / mixed-batch operators: argument
// validation and launches.  Nothing here allocates or synchronises.
#include <cmath>
#include <cstring>

#include "gdnr_device.cuh"
#include "gdnr_hybrid.h"

using namespace gdnr;

namespace gdnr {

int multiprocessor_count() {
  static std::atomic<int> count[DynSmemCache::kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 1;
  const bool cached = dev >= 0 && dev < DynSmemCache::kMaxDevices;
  int n = cached ? count[dev].load(std::memory_order_relaxed) : 0;
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) return 1;
    if (cached) count[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

cudaError_t encode_bf16_map(CUtensorMap* map, const void* base, int rank, const uint64_t* dims, const uint64_t* strides,
                            const uint32_t* box) {
  static std::atomic<EncodeFn> fn{nullptr};
  EncodeFn enc = fn.load(std::memory_order_acquire);
  if (!enc) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return cudaErrorNotSupported;
    enc = reinterpret_cast<EncodeFn>(ptr);
    fn.store(enc, std::memory_order_release);
  }
  const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
  const CUresult rc = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, strides, box, ones,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return rc == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

}  // namespace gdnr

namespace {

const int HY_BF16[] = {GDNR_BF16};
const int HY_F32[] = {GDNR_F32};
const int HY_I32[] = {GDNR_I32};
const int HY_U8[] = {GDNR_U8};
const int HY_GATE[] = {GDNR_F32, GDNR_BF16, GDNR_F16};
const int HY_WEIGHT[] = {GDNR_BF16, GDNR_F32};

#define CHECK(expr)                 \
  do {                              \
    int _rc = (expr);               \
    if (_rc != GDNR_OK) return _rc; \
  } while (0)

// Token and page counts are int32 in the kernels, so are products of heads.
constexpr int64_t MAX_EXTENT = int64_t(1) << 30;

int check_extents(const gdnr_tensor& t, const char* name) {
  for (int i = 0; i < t.ndim; ++i)
    if (t.shape[i] > MAX_EXTENT) return set_error(GDNR_ERR_UNSUPPORTED, "%s: dim %d above 2^30", name, i);
  return GDNR_OK;
}

// A row-gathered bf16 tensor: innermost contiguous, base and outer strides 16-byte multiples.
int check_rows(const gdnr_tensor& t, const char* name, int ndim, const int64_t* want) {
  CHECK(check_tensor(t, name, ndim, HY_BF16, 1, want));
  CHECK(check_extents(t, name));
  CHECK(check_inner_contiguous(t, name));
  return check_aligned16(t, name, 0);
}

// overlaps(), of tensors that have elements (an empty one has no address of its own)
bool touches(const gdnr_tensor& a, const gdnr_tensor& b) {
  for (int i = 0; i < a.ndim; ++i)
    if (a.shape[i] == 0) return false;
  for (int i = 0; i < b.ndim; ++i)
    if (b.shape[i] == 0) return false;
  return overlaps(a, b);
}

// log2 of a power of two, -1 of anything else
int shift_of(int64_t x) {
  for (int s = 0; s < 31; ++s)
    if (x == (int64_t(1) << s)) return s;
  return -1;
}

// cu_seqlens [N+1]; N out
int check_seqlens(const gdnr_tensor& t, int64_t* n) {
  CHECK(check_tensor(t, "cu_seqlens", 1, HY_I32, 1, nullptr));
  CHECK(check_inner_contiguous(t, "cu_seqlens"));
  if (t.shape[0] < 1) return set_error(GDNR_ERR_ARG, "cu_seqlens: needs N + 1 entries, got none");
  if (t.shape[0] > (1 << 20)) return set_error(GDNR_ERR_UNSUPPORTED, "cu_seqlens: more than 2^20 sequences");
  *n = t.shape[0] - 1;
  return GDNR_OK;
}

}  // namespace

extern "C" {

int gdnr_gdn_prefill(const gdnr_prefill_args* x, void* stream) {
  if (!x) return set_error(GDNR_ERR_ARG, "args: null pointer");
  PrefillParams p;
  memset(&p, 0, sizeof(p));
  int64_t n = 0;
  CHECK(check_seqlens(x->cu_seqlens, &n));
  CHECK(check_tensor(x->state, "state", 4, HY_F32, 1, nullptr));
  const int64_t S = x->state.shape[0], HV = x->state.shape[1], V = x->state.shape[2], K = x->state.shape[3];
  if (K != 128 || V != 128)
    return set_error(GDNR_ERR_UNSUPPORTED, "state: head dims V=%lld K=%lld: only K = V = 128 is implemented", (long long)V,
                     (long long)K);
  if (HV < 1 || HV > 4096 || S > MAX_EXTENT) return set_error(GDNR_ERR_UNSUPPORTED, "state: HV outside [1, 4096] or too many slots");
  if (x->state.stride[3] != 1 || x->state.stride[2] != K)
    return set_error(GDNR_ERR_LAYOUT, "state: rows of one head must be packed (strides K, 1 of the last two dims)");
  CHECK(check_aligned16(x->state, "state", 0));
  CHECK(check_tensor(x->mixed_qkv, "mixed_qkv", 2, HY_BF16, 1, nullptr));
  CHECK(check_extents(x->mixed_qkv, "mixed_qkv"));
  const int64_t T = x->mixed_qkv.shape[0], W = x->mixed_qkv.shape[1];
  const int64_t rest = W - HV * V;
  if (rest < 2 * K || rest % (2 * K))
    return set_error(GDNR_ERR_ARG, "mixed_qkv: width %lld is not 2*H*128 + HV*128 for HV=%lld", (long long)W, (long long)HV);
  const int64_t H = rest / (2 * K);
  if (HV % H) return set_error(GDNR_ERR_ARG, "HV=%lld is not a multiple of H=%lld", (long long)HV, (long long)H);
  CHECK(check_inner_contiguous(x->mixed_qkv, "mixed_qkv"));
  CHECK(check_aligned16(x->mixed_qkv, "mixed_qkv", 0));
  const int64_t want_ab[2] = {T, HV}, want_hv[1] = {HV}, want_n[1] = {n};
  CHECK(check_tensor(x->a, "a", 2, HY_GATE, 3, want_ab));
  CHECK(check_tensor(x->b, "b", 2, HY_GATE, 3, want_ab));
  CHECK(check_tensor(x->a_log, "A_log", 1, HY_F32, 1, want_hv));
  CHECK(check_tensor(x->dt_bias, "dt_bias", 1, HY_F32, 1, want_hv));
  const int64_t want_o[3] = {T, HV, V};
  CHECK(check_rows(x->out, "out", 3, want_o));
  if (present(x->state_indices)) {
    CHECK(check_tensor(x->state_indices, "state_indices", 1, HY_I32, 1, want_n));
    p.sidx = static_cast<const int32_t*>(x->state_indices.data);
    p.si_s = x->state_indices.stride[0];
  } else if (S < n) {
    return set_error(GDNR_ERR_ARG, "state: %lld slots for %lld sequences", (long long)S, (long long)n);
  }
  if (present(x->has_initial)) {
    CHECK(check_tensor(x->has_initial, "has_initial", 1, HY_U8, 1, want_n));
    p.has_init = static_cast<const uint8_t*>(x->has_initial.data);
    p.hi_s = x->has_initial.stride[0];
  }
  if (x->max_seqlen < 0) return set_error(GDNR_ERR_ARG, "max_seqlen must not be negative");
  if (touches(x->out, x->mixed_qkv) || touches(x->out, x->state))
    return set_error(GDNR_ERR_ALIAS, "out must not overlap mixed_qkv or state");
  if (touches(x->state, x->mixed_qkv)) return set_error(GDNR_ERR_ALIAS, "state must not overlap mixed_qkv");
  p.mixed = static_cast<const uint16_t*>(x->mixed_qkv.data);
  p.mx_s = x->mixed_qkv.stride[0];
  p.a = x->a.data;
  p.a_st = x->a.stride[0], p.a_sh = x->a.stride[1], p.a_dt = x->a.dtype;
  p.b = x->b.data;
  p.b_st = x->b.stride[0], p.b_sh = x->b.stride[1], p.b_dt = x->b.dtype;
  p.a_log = static_cast<const float*>(x->a_log.data);
  p.al_s = x->a_log.stride[0];
  p.dt_bias = static_cast<const float*>(x->dt_bias.data);
  p.db_s = x->dt_bias.stride[0];
  p.state = static_cast<float*>(x->state.data);
  p.st_ss = x->state.stride[0], p.st_sh = x->state.stride[1];
  p.cu = static_cast<const int32_t*>(x->cu_seqlens.data);
  p.out = static_cast<uint16_t*>(x->out.data);
  p.o_st = x->out.stride[0], p.o_sh = x->out.stride[1];
  p.N = int(n), p.H = int(H), p.HV = int(HV), p.S = int(S), p.T = int(T);
  p.err = x->error_flag ? x->error_flag : default_error_word();
  if (!p.err) return set_error(GDNR_ERR_CUDA, "no device error word available");
  if (n == 0) return GDNR_OK;
  if (n * HV > (int64_t(1) << 28)) return set_error(GDNR_ERR_UNSUPPORTED, "N * HV above 2^28");
  const int64_t need = prefill_workspace_bytes(T, n, HV, x->max_seqlen);
  p.images = static_cast<uint8_t*>(x->workspace);
  if (need > 0 && (!p.images || reinterpret_cast<uintptr_t>(p.images) % 16 || x->workspace_bytes < need))
    return set_error(GDNR_ERR_ARG, "workspace: needs %lld bytes at a 16-byte aligned address", (long long)need);
  if ((T / 64 + n) * H > (int64_t(1) << 30)) return set_error(GDNR_ERR_UNSUPPORTED, "T / 64 * H above 2^30");
  return cuda_status(launch_prefill(p, x->max_seqlen, static_cast<cudaStream_t>(stream)), "gdnr_gdn_prefill launch");
}

int64_t gdnr_gdn_prefill_workspace(int64_t tokens, int64_t sequences, int32_t value_heads, int32_t max_seqlen) {
  return prefill_workspace_bytes(tokens, sequences, value_heads, max_seqlen);
}

int gdnr_qk_norm_rope_append(const gdnr_append_args* x, void* stream) {
  if (!x) return set_error(GDNR_ERR_ARG, "args: null pointer");
  AppendParams p;
  memset(&p, 0, sizeof(p));
  CHECK(check_rows(x->q, "q", 3, nullptr));
  const int64_t T = x->q.shape[0], Hq = x->q.shape[1], D = x->q.shape[2];
  if (D != 64 && D != 128 && D != 256)
    return set_error(GDNR_ERR_UNSUPPORTED, "head dim %lld: only 64, 128 and 256 are implemented", (long long)D);
  const int64_t any_k[3] = {T, -1, D};
  CHECK(check_rows(x->k, "k", 3, any_k));
  const int64_t Hk = x->k.shape[1];
  const int64_t want_k[3] = {T, Hk, D}, want_q[3] = {T, Hq, D}, want_t[1] = {T}, want_d[1] = {D};
  CHECK(check_rows(x->v, "v", 3, want_k));
  CHECK(check_rows(x->q_out, "q_out", 3, want_q));
  if (Hq > 65535 || Hk > 65535) return set_error(GDNR_ERR_UNSUPPORTED, "more than 65535 heads");
  if (present(x->q_weight)) {
    CHECK(check_tensor(x->q_weight, "q_weight", 1, HY_WEIGHT, 2, want_d));
    CHECK(check_inner_contiguous(x->q_weight, "q_weight"));
    CHECK(check_aligned16(x->q_weight, "q_weight", 0));
    p.qw = x->q_weight.data, p.qw_dt = x->q_weight.dtype;
  }
  if (present(x->k_weight)) {
    CHECK(check_tensor(x->k_weight, "k_weight", 1, HY_WEIGHT, 2, want_d));
    CHECK(check_inner_contiguous(x->k_weight, "k_weight"));
    CHECK(check_aligned16(x->k_weight, "k_weight", 0));
    p.kw = x->k_weight.data, p.kw_dt = x->k_weight.dtype;
  }
  CHECK(check_tensor(x->positions, "positions", 1, HY_I32, 1, want_t));
  CHECK(check_tensor(x->slots, "slots", 1, HY_I32, 1, want_t));
  CHECK(check_tensor(x->cos_sin, "cos_sin", 2, HY_F32, 1, nullptr));
  CHECK(check_extents(x->cos_sin, "cos_sin"));
  CHECK(check_inner_contiguous(x->cos_sin, "cos_sin"));
  const int64_t rot = x->cos_sin.shape[1];
  if (rot > D || rot % 2) return set_error(GDNR_ERR_ARG, "cos_sin: width %lld must be even and at most D=%lld", (long long)rot, (long long)D);
  const int64_t any_c[4] = {-1, -1, Hk, D};
  CHECK(check_rows(x->k_cache, "k_cache", 4, any_c));
  const int64_t pages = x->k_cache.shape[0], ps = x->k_cache.shape[1];
  const int64_t want_c[4] = {pages, ps, Hk, D};
  CHECK(check_rows(x->v_cache, "v_cache", 4, want_c));
  if (ps < 1) return set_error(GDNR_ERR_ARG, "k_cache: page_size must be at least 1");
  if (!(x->eps >= 0.f) || !std::isfinite(x->weight_offset)) return set_error(GDNR_ERR_ARG, "eps or weight_offset out of range");
  if (x->interleaved != 0 && x->interleaved != 1) return set_error(GDNR_ERR_ARG, "interleaved must be 0 or 1");
  const bool same_q = x->q.data == x->q_out.data && x->q.stride[0] == x->q_out.stride[0] && x->q.stride[1] == x->q_out.stride[1];
  if (!same_q && touches(x->q, x->q_out)) return set_error(GDNR_ERR_ALIAS, "q_out must be q itself or not overlap it");
  if (touches(x->k_cache, x->v_cache) && x->k_cache.data == x->v_cache.data)
    return set_error(GDNR_ERR_ALIAS, "k_cache and v_cache are the same buffer");
  p.q = static_cast<const uint16_t*>(x->q.data), p.q_st = x->q.stride[0], p.q_sh = x->q.stride[1];
  p.k = static_cast<const uint16_t*>(x->k.data), p.k_st = x->k.stride[0], p.k_sh = x->k.stride[1];
  p.v = static_cast<const uint16_t*>(x->v.data), p.v_st = x->v.stride[0], p.v_sh = x->v.stride[1];
  p.pos = static_cast<const int32_t*>(x->positions.data), p.pos_s = x->positions.stride[0];
  p.slots = static_cast<const int32_t*>(x->slots.data), p.sl_s = x->slots.stride[0];
  p.table = static_cast<const float*>(x->cos_sin.data), p.tb_s = x->cos_sin.stride[0];
  p.q_out = static_cast<uint16_t*>(x->q_out.data), p.qo_st = x->q_out.stride[0], p.qo_sh = x->q_out.stride[1];
  p.kc = static_cast<uint16_t*>(x->k_cache.data);
  p.kc_sp = x->k_cache.stride[0], p.kc_st = x->k_cache.stride[1], p.kc_sh = x->k_cache.stride[2];
  p.vc = static_cast<uint16_t*>(x->v_cache.data);
  p.vc_sp = x->v_cache.stride[0], p.vc_st = x->v_cache.stride[1], p.vc_sh = x->v_cache.stride[2];
  p.T = int(T), p.Hq = int(Hq), p.Hk = int(Hk), p.D = int(D), p.rot = int(rot), p.P = int(x->cos_sin.shape[0]);
  p.pages = int(pages), p.page_size = int(ps), p.inter = x->interleaved;
  p.page_shift = shift_of(ps);
  p.tb_vec = reinterpret_cast<uintptr_t>(p.table) % 16 == 0 && p.tb_s % 4 == 0 && (rot / 2) % 8 == 0;
  p.eps = x->eps, p.w_off = x->weight_offset;
  p.err = x->error_flag ? x->error_flag : default_error_word();
  if (!p.err) return set_error(GDNR_ERR_CUDA, "no device error word available");
  if (T == 0 || Hq + Hk == 0) return GDNR_OK;
  if (T * (Hq + 2 * Hk) > (int64_t(1) << 31)) return set_error(GDNR_ERR_UNSUPPORTED, "T * heads above 2^31");
  return cuda_status(launch_append(p, static_cast<cudaStream_t>(stream)), "gdnr_qk_norm_rope_append launch");
}

int64_t gdnr_paged_attention_workspace(int32_t head_dim) { return attn_workspace_bytes(head_dim); }

int gdnr_paged_attention(const gdnr_attn_args* x, void* stream) {
  if (!x) return set_error(GDNR_ERR_ARG, "args: null pointer");
  AttnParams p;
  memset(&p, 0, sizeof(p));
  CHECK(check_rows(x->q, "q", 3, nullptr));
  const int64_t T = x->q.shape[0], Hq = x->q.shape[1], D = x->q.shape[2];
  if (D != 64 && D != 128 && D != 256)
    return set_error(GDNR_ERR_UNSUPPORTED, "head dim %lld: only 64, 128 and 256 are implemented", (long long)D);
  const int64_t any_c[4] = {-1, -1, -1, D};
  CHECK(check_rows(x->k_cache, "k_cache", 4, any_c));
  const int64_t pages = x->k_cache.shape[0], ps = x->k_cache.shape[1], Hk = x->k_cache.shape[2];
  const int64_t want_c[4] = {pages, ps, Hk, D};
  CHECK(check_rows(x->v_cache, "v_cache", 4, want_c));
  if (ps < 1) return set_error(GDNR_ERR_ARG, "k_cache: page_size must be at least 1");
  if (Hk < 1 || Hq < 1 || Hq % Hk) return set_error(GDNR_ERR_ARG, "Hq=%lld is not a multiple of Hk=%lld", (long long)Hq, (long long)Hk);
  if (Hq > 4096) return set_error(GDNR_ERR_UNSUPPORTED, "more than 4096 query heads");
  int64_t n = 0;
  CHECK(check_seqlens(x->cu_seqlens, &n));
  const int64_t want_b[2] = {n, -1}, want_n[1] = {n}, want_q[3] = {T, Hq, D}, want_l[2] = {T, Hq};
  CHECK(check_tensor(x->block_table, "block_table", 2, HY_I32, 1, want_b));
  CHECK(check_extents(x->block_table, "block_table"));
  CHECK(check_inner_contiguous(x->block_table, "block_table"));
  CHECK(check_tensor(x->kv_lens, "kv_lens", 1, HY_I32, 1, want_n));
  CHECK(check_rows(x->out, "out", 3, want_q));
  if (present(x->lse)) {
    CHECK(check_tensor(x->lse, "lse", 2, HY_F32, 1, want_l));
    p.lse = static_cast<float*>(x->lse.data), p.l_st = x->lse.stride[0], p.l_sh = x->lse.stride[1];
  }
  if (!std::isfinite(x->scale)) return set_error(GDNR_ERR_ARG, "scale must be finite");
  if (x->max_seqlen < 0) return set_error(GDNR_ERR_ARG, "max_seqlen must not be negative");
  if (touches(x->out, x->q) || touches(x->out, x->k_cache) || touches(x->out, x->v_cache))
    return set_error(GDNR_ERR_ALIAS, "out must not overlap q or the caches");
  if (T * (Hq / Hk) > MAX_EXTENT) return set_error(GDNR_ERR_UNSUPPORTED, "T * Hq/Hk above 2^30");
  p.q = static_cast<const uint16_t*>(x->q.data), p.q_st = x->q.stride[0], p.q_sh = x->q.stride[1];
  p.k = static_cast<const uint16_t*>(x->k_cache.data);
  p.k_sp = x->k_cache.stride[0], p.k_st = x->k_cache.stride[1], p.k_sh = x->k_cache.stride[2];
  p.v = static_cast<const uint16_t*>(x->v_cache.data);
  p.v_sp = x->v_cache.stride[0], p.v_st = x->v_cache.stride[1], p.v_sh = x->v_cache.stride[2];
  p.table = static_cast<const int32_t*>(x->block_table.data), p.tb_s = x->block_table.stride[0];
  p.kv_lens = static_cast<const int32_t*>(x->kv_lens.data), p.kl_s = x->kv_lens.stride[0];
  p.cu = static_cast<const int32_t*>(x->cu_seqlens.data);
  p.out = static_cast<uint16_t*>(x->out.data), p.o_st = x->out.stride[0], p.o_sh = x->out.stride[1];
  p.scale = x->scale;
  p.N = int(n), p.T = int(T), p.Hq = int(Hq), p.Hk = int(Hk), p.G = int(Hq / Hk), p.D = int(D);
  p.pages = int(pages), p.page_size = int(ps), p.width = int(x->block_table.shape[1]);
  p.page_shift = shift_of(ps);
  // row * (G magic - 2^32) has to stay below 2^32 for rows up to T * G
  if (p.G > 1 && T * p.G * p.G < (int64_t(1) << 32)) p.g_magic = uint32_t(((int64_t(1) << 32) + p.G - 1) / p.G);
  p.max_q = x->max_seqlen > 0 ? x->max_seqlen : int(T);
  p.err = x->error_flag ? x->error_flag : default_error_word();
  if (!p.err) return set_error(GDNR_ERR_CUDA, "no device error word available");
  if (n == 0 || T == 0) return GDNR_OK;
  p.ws = static_cast<float*>(x->workspace);
  p.ws_bytes = x->workspace_bytes;
  if (!p.ws || reinterpret_cast<uintptr_t>(p.ws) % 16 || p.ws_bytes < attn_workspace_bytes(int(D)))
    return set_error(GDNR_ERR_ARG, "workspace: needs %lld bytes at a 16-byte aligned address", (long long)attn_workspace_bytes(int(D)));
  return cuda_status(launch_attn(p, static_cast<cudaStream_t>(stream)), "gdnr_paged_attention launch");
}

}  // extern "C"
