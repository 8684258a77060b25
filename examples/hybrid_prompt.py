"""A hybrid block (one GDN layer, one softmax-attention layer) from prompts to generated tokens.

    python examples/hybrid_prompt.py

Prompts of different lengths run packed through both layers: ``gdn_prefill`` leaves each
sequence's float32 state, which is handed to the decode step's ``ReplayState`` (FP8 checkpoint + ring);
``qk_norm_rope_append`` and ``paged_attention`` fill and read the paged cache.  Tokens then go one
at a time: ``ReplayState.step`` for the GDN layer, the same two calls for the attention layer.
Weights are random; the point is which call gets what.
"""

from __future__ import annotations

import pathlib
import sys
from dataclasses import dataclass

import torch

ROOT = pathlib.Path(__file__).resolve().parent.parent
if str(ROOT / "fp8-replayssm-gdn-kernel_b200") not in sys.path:
    sys.path.insert(0, str(ROOT / "fp8-replayssm-gdn-kernel_b200"))

import gdnr  # noqa: E402

BF16 = torch.bfloat16


@dataclass
class Sizes:
    width: int = 512  # of the residual stream
    key_heads: int = 4  # GDN layer, head dim 128
    value_heads: int = 8
    q_heads: int = 8  # attention layer
    kv_heads: int = 2
    head_dim: int = 128
    rot_dim: int = 32  # a quarter of the head is rotated
    page: int = 64
    pages_per_seq: int = 8


class HybridBlock:
    """x + GDN(x), then + attention; random weights."""

    def __init__(self, sizes: Sizes, seed: int = 0, device: str = "cuda"):
        self.s = s = sizes
        g = torch.Generator(device=device)
        g.manual_seed(seed)

        def w(rows, cols):
            return (torch.randn(rows, cols, generator=g, device=device) * rows ** -0.5).to(BF16)

        self.w_qkv = w(s.width, 2 * s.key_heads * 128 + s.value_heads * 128)
        self.w_ab = w(s.width, 2 * s.value_heads)
        self.w_gdn_out = w(s.value_heads * 128, s.width)
        self.a_log = torch.log(1 + 15 * torch.rand(s.value_heads, generator=g, device=device))
        self.dt_bias = 0.5 * torch.randn(s.value_heads, generator=g, device=device)
        self.w_attn = w(s.width, (s.q_heads + 2 * s.kv_heads) * s.head_dim)
        self.w_attn_out = w(s.q_heads * s.head_dim, s.width)
        self.q_norm = torch.ones(s.head_dim, dtype=BF16, device=device)
        self.k_norm = torch.ones(s.head_dim, dtype=BF16, device=device)
        self.table = gdnr.rope_table(s.page * s.pages_per_seq, s.rot_dim, device=device)

    def gdn_inputs(self, x):
        a, b = (x @ self.w_ab).split(self.s.value_heads, -1)
        return x @ self.w_qkv, a, b

    def attention(self, x, cache, positions, cu_seqlens, kv_lens, max_seqlen):
        """Norm, rotate and append the tokens of every sequence, then attend; cu_seqlens packs them."""
        s = self.s
        q, k, v = (x @ self.w_attn).split([s.q_heads * s.head_dim, s.kv_heads * s.head_dim, s.kv_heads * s.head_dim], -1)
        n = len(x)
        seq = torch.searchsorted(cu_seqlens[1:].contiguous(), torch.arange(n, device=x.device, dtype=torch.int32), right=True)
        slots = cache.block_table[seq, positions // s.page] * s.page + positions % s.page
        q = gdnr.qk_norm_rope_append(q.unflatten(-1, (s.q_heads, -1)), k.unflatten(-1, (s.kv_heads, -1)), v.unflatten(-1, (s.kv_heads, -1)),
                                     positions, slots.int(), self.table, cache.k, cache.v, q_weight=self.q_norm, k_weight=self.k_norm)
        o = gdnr.paged_attention(q, cache.k, cache.v, cache.block_table, kv_lens, cu_seqlens, max_seqlen=max_seqlen)
        return o.flatten(1) @ self.w_attn_out


class PagedCache:
    def __init__(self, sizes: Sizes, sequences: int, device: str = "cuda"):
        pages = sequences * sizes.pages_per_seq
        shape = (pages, sizes.page, sizes.kv_heads, sizes.head_dim)
        self.k, self.v = (torch.empty(shape, dtype=BF16, device=device) for _ in range(2))
        self.block_table = torch.randperm(pages, device=device).int().view(sequences, -1)


def prefill(block: HybridBlock, x, lens, cache):
    """All prompts at once: x [T, width] packed; returns the outputs and the GDN states [N,HV,128,128]."""
    dev = x.device
    cu = torch.tensor([0] + list(lens), device=dev).cumsum(0).int()
    state = torch.empty(len(lens), block.s.value_heads, 128, 128, device=dev)
    o = gdnr.gdn_prefill(*block.gdn_inputs(x), block.a_log, block.dt_bias, state, cu,
                         has_initial_state=torch.zeros(len(lens), dtype=torch.bool, device=dev), max_seqlen=max(lens))
    x = x + o.flatten(1) @ block.w_gdn_out
    positions = torch.cat([torch.arange(m, device=dev) for m in lens]).int()
    kv_lens = torch.tensor(lens, dtype=torch.int32, device=dev)
    return x + block.attention(x, cache, positions, cu, kv_lens, max(lens)), state


def decode(block: HybridBlock, x, replay: gdnr.ReplayState, cache, kv_lens):
    """One token of each sequence: x [N, width]; advances the replay state and kv_lens."""
    n, dev = len(x), x.device
    advanced = torch.empty_like(replay.pos)
    o = replay.step(*block.gdn_inputs(x), block.a_log, block.dt_bias, pos_out=advanced)
    replay.pos.copy_(advanced)
    x = x + o.flatten(1) @ block.w_gdn_out
    positions = kv_lens.clone()
    kv_lens += 1
    return x + block.attention(x, cache, positions, torch.arange(n + 1, device=dev, dtype=torch.int32), kv_lens, 1)


def main() -> None:
    sizes, lens, new = Sizes(), [37, 1, 200, 129], 20
    block, cache = HybridBlock(sizes), PagedCache(sizes, len(lens))
    x = torch.randn(sum(lens), sizes.width, device="cuda").to(BF16)
    out, state = prefill(block, x, lens, cache)
    replay = gdnr.ReplayState.allocate(len(lens), sizes.key_heads, sizes.value_heads, ring_len=16)
    replay.load_state(state)
    kv_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    last = out[torch.tensor(lens, device="cuda").cumsum(0) - 1]
    for _ in range(new):  # the block's own output stands in for the next token's embedding
        last = decode(block, torch.nn.functional.normalize(last.float(), dim=-1).mul(sizes.width ** 0.5).to(BF16), replay, cache, kv_lens)
    torch.cuda.synchronize()
    if gdnr.read_device_error():
        raise SystemExit("device error word set")
    print(f"{sum(lens)} prompt tokens in {len(lens)} sequences, {new} tokens each; |x| {float(last.float().norm(dim=-1).mean()):.3f}")


if __name__ == "__main__":
    main()
