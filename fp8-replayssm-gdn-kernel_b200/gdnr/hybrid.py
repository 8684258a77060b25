"""Prompts and mixed batches of a hybrid model (GDN layers and softmax-attention layers).

The decode step of :mod:`gdnr.ops` starts from a state that something has to
have built from the prompt, and a hybrid model's other layers attend a paged cache:

* :func:`gdn_prefill` -- the gated delta rule over a ragged batch: whole
  prompts, continued prompts, a few tokens to verify, or one token each, on a float32 state;
* :func:`qk_norm_rope_append` -- per-head RMS norm of queries and keys, rotary
  positions and the append of keys and values to a paged cache;
* :func:`paged_attention` -- causal attention of the new tokens over that cache.

A ragged batch is packed: the tokens of sequence ``n`` are rows ``cu_seqlens[n]``
to ``cu_seqlens[n + 1] - 1``; rows that belong to no sequence are not written.  ``max_seqlen`` is
the longest sequence as far as the host knows it (it picks kernels and grids; ``paged_attention``
reports a longer one in the device error word as ``GDNR_DEVERR_BAD_HINT``).  All work runs on the current stream of the
tensors' device; nothing synchronises.
"""

from __future__ import annotations

import math
import struct

import torch

from . import _lib
from .ops import _err_ptr

_PREFILL_TAIL = struct.Struct("@iiPqP")
_APPEND_TAIL = struct.Struct("@ffiiP")
_ATTN_TAIL = struct.Struct("@fiPqP")


def _err(error_flag) -> int:
    return _err_ptr(error_flag) or 0


def gdn_prefill(
    mixed_qkv: torch.Tensor,
    a: torch.Tensor,
    b: torch.Tensor,
    A_log: torch.Tensor,
    dt_bias: torch.Tensor,
    state: torch.Tensor,
    cu_seqlens: torch.Tensor,
    *,
    state_indices: torch.Tensor | None = None,
    has_initial_state: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    max_seqlen: int = 0,
    error_flag: torch.Tensor | None = None,
) -> torch.Tensor:
    """Run every sequence's tokens through a GDN layer's recurrence; returns ``out`` [T,HV,V] bf16.

    ``mixed_qkv`` [T, 2*H*K + HV*V] bf16, ``a``/``b`` [T,HV], ``A_log``/``dt_bias`` [HV]
    float32 as the decode step takes them.  ``state`` [slots,HV,V,K] float32 is
    updated in place: sequence ``n`` continues slot ``state_indices[n]`` (slot ``n`` without it),
    or starts from zeros where ``has_initial_state[n]`` is false.  An index ``<= 0`` is the
    null slot (``out`` rows are zeros, no state is touched), one past the pool likewise, reported as
    ``GDNR_DEVERR_BAD_SLOT``; the others must be distinct.  An empty sequence leaves its
    state as it is (zeros if it starts from zeros).

    ``max_seqlen`` (the mean length where it is 0) decides for the whole call: up to 20 tokens token by
    token, else in chunks of 64, with a workspace of 21568 bytes for each of the ``T // 64 + N`` chunks of
    each value head.  Many single tokens beside a long prompt are better off in a call of their own.

    The state can be handed to the decode step with :meth:`gdnr.ReplayState.load_state`.
    """
    if out is None:
        out = mixed_qkv.new_empty((mixed_qkv.shape[0], state.shape[1], state.shape[2]), dtype=torch.bfloat16)
    nbytes = _lib.load().gdnr_gdn_prefill_workspace(mixed_qkv.shape[0], cu_seqlens.shape[0] - 1, state.shape[1], max_seqlen)
    workspace = mixed_qkv.new_empty(nbytes, dtype=torch.uint8) if nbytes > 0 else None
    _lib.call_tensors("gdnr_gdn_prefill", (mixed_qkv, a, b, A_log, dt_bias, state, cu_seqlens, state_indices, has_initial_state, out),
                      _PREFILL_TAIL.pack(max_seqlen, 0, workspace.data_ptr() if nbytes > 0 else 0, nbytes, _err(error_flag)))
    return out


def qk_norm_rope_append(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    positions: torch.Tensor,
    slots: torch.Tensor,
    cos_sin: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    *,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    weight_offset: float = 0.0,
    interleaved: bool = False,
    q_out: torch.Tensor | None = None,
    error_flag: torch.Tensor | None = None,
) -> torch.Tensor:
    """Norm, rotate and append one layer's new tokens; returns the queries [T,Hq,D] bf16.

    ``q`` [T,Hq,D], ``k``/``v`` [T,Hk,D] bf16 (views of a packed projection do; D = 64, 128 or
    256).  With a weight [D] (bf16 or float32) each head is divided by its root mean square
    and multiplied by ``weight + weight_offset``.  The first ``cos_sin.shape[1]`` elements are
    rotated by row ``positions[t]`` of ``cos_sin`` (see :func:`rope_table`).  ``k``
    and ``v`` go to row ``slots[t] % page_size`` of page ``slots[t] // page_size`` of the caches
    [pages,page_size,Hk,D]; a negative slot is padding.  ``q_out`` may be ``q`` itself.
    """
    if q_out is None:
        q_out = q.new_empty(q.shape)
    _lib.call_tensors("gdnr_qk_norm_rope_append", (q, k, v, q_weight, k_weight, positions, slots, cos_sin, q_out, k_cache, v_cache),
                      _APPEND_TAIL.pack(eps, weight_offset, 1 if interleaved else 0, 0, _err(error_flag)))
    return q_out


def paged_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    kv_lens: torch.Tensor,
    cu_seqlens: torch.Tensor,
    *,
    scale: float | None = None,
    out: torch.Tensor | None = None,
    return_lse: bool = False,
    max_seqlen: int = 0,
    error_flag: torch.Tensor | None = None,
):
    """Causal attention of each sequence's new tokens over its pages; returns ``out`` [T,Hq,D] bf16.

    The ``m`` new tokens of sequence ``n`` are the last of its ``kv_lens[n]`` cached ones (append
    them first): row ``i`` attends places ``0 .. kv_lens[n] - m + i``; a row without any
    is zeros.  ``k_cache``/``v_cache`` [pages,page_size,Hk,D] bf16, any page size; ``block_table``
    [N,width] int32 holds each sequence's pages; a page outside the cache, or a length outside
    ``[0, width * page_size]``, is reported as ``GDNR_DEVERR_BAD_SLOT``.  ``scale`` defaults to ``D ** -0.5``.  With
    ``return_lse`` also the float32 log of each row's sum of exponentials [T,Hq]
    (-inf for a row without places).
    """
    head_dim = q.shape[-1]
    if out is None:
        out = q.new_empty(q.shape)
    lse = q.new_empty(q.shape[:2], dtype=torch.float32) if return_lse else None
    nbytes = _workspace_bytes(q.get_device(), head_dim)
    workspace = q.new_empty(nbytes, dtype=torch.uint8)
    _lib.call_tensors("gdnr_paged_attention", (q, k_cache, v_cache, block_table, kv_lens, cu_seqlens, out, lse),
                      _ATTN_TAIL.pack(head_dim ** -0.5 if scale is None else scale, max_seqlen, workspace.data_ptr(), nbytes,
                                      _err(error_flag)))
    return (out, lse) if return_lse else out


_workspace: dict[tuple[int, int], int] = {}


def _workspace_bytes(device_index: int, head_dim: int) -> int:
    n = _workspace.get((device_index, head_dim))
    if n is None:
        with torch.cuda.device(device_index):
            n = int(_lib.load().gdnr_paged_attention_workspace(head_dim))
        _workspace[(device_index, head_dim)] = n
    return n


def rope_table(positions: int, rot_dim: int, base: float = 10000.0, *, scaling: str = "none", factor: float = 1.0,
               original_positions: int = 0, beta_fast: float = 32.0, beta_slow: float = 1.0,
               device: torch.device | str = "cuda") -> torch.Tensor:
    """cos and sin of the rotary angles, [positions, rot_dim] float32 (cos of rot_dim/2 angles, then sin).

    ``scaling`` for contexts longer than the trained one: "none"; "linear" (positions divided by
    ``factor``); or "yarn" (YaRN, Peng et al. 2023): an angle that turns more than ``beta_fast``
    times over the ``original_positions`` keeps its frequency, one that turns less than
    ``beta_slow`` times is divided by ``factor``, linearly blended in between, and cos and sin
    are multiplied by 0.1 ln(factor) + 1.  Angles are taken in float64.
    """
    if rot_dim <= 0 or rot_dim % 2:
        raise ValueError(f"rot_dim must be positive and even (got {rot_dim})")
    if scaling not in ("none", "linear", "yarn"):
        raise ValueError(f"scaling must be 'none', 'linear' or 'yarn' (got {scaling!r})")
    if factor < 1.0 or (scaling == "yarn" and original_positions <= 0):
        raise ValueError("factor must be at least 1, and 'yarn' needs original_positions")
    index = torch.arange(0, rot_dim, 2, dtype=torch.float64)
    freq = base ** (-index / rot_dim)
    gain = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        def place(turns):  # the (fractional) pair index whose angle turns so often over the trained positions
            return rot_dim * math.log(original_positions / (turns * 2 * math.pi)) / (2 * math.log(base))

        low, high = max(math.floor(place(beta_fast)), 0), min(math.ceil(place(beta_slow)), rot_dim - 1)
        ramp = ((torch.arange(rot_dim // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
        freq = freq * (1 - ramp) + freq / factor * ramp
        gain = 0.1 * math.log(factor) + 1.0
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * freq
    return (gain * torch.cat([angle.cos(), angle.sin()], 1)).to(torch.float32).to(device)
