"""Cases of the prompt and mixed-batch operators of a hybrid (Gated DeltaNet + attention) model.

Three operators are measured, over the ranges a serving process meets:

* ``gdn``: the gated delta rule over a ragged batch of sequences (``gdnr.gdn_prefill``): whole
  prompts, continued prompts, a few tokens to verify, and single tokens, on a float32 state pool;
* ``append``: per-head RMS norm of queries and keys, rotary positions and the append to a paged
  cache in one call (``gdnr.qk_norm_rope_append``);
* ``attn``: causal attention of each sequence's new tokens over its paged cache
  (``gdnr.paged_attention``): single tokens, chunks of a prompt, and both in one batch.

With ``own`` false, ``run`` computes them with elementary torch operations in float32, rounded once
at the end; with ``own`` true it calls the package.  Lengths are texts ("17,1,300"): one per sequence.
"""

import math
import os
import sys

import torch

own = False

DEV = "cuda"
EPS = 1e-6  # of the L2 norm of the delta rule's keys and of the RMS norm


def _package():
    root = os.path.join(os.getcwd(), "fp8-replayssm-gdn-kernel_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import gdnr

    return gdnr


def _lens(text):
    return [int(x) for x in text.split(",")]


def _text(values):
    return ",".join(str(int(v)) for v in values)


# ------------------------------------------------------------------------------------------ cases
def listed():
    import random

    r = random.Random(20)
    decode_ctx = [r.randint(100, 8000) for _ in range(64)]
    return [
        # one sequence generating one token: latency of the smallest call
        dict(name="gdn_token_b1", op="gdn", h=16, hv=32, lens="1", fresh=False),
        # the repository's batch of 64 sequences, one token each, on a float32 state
        dict(name="gdn_token_b64", op="gdn", h=16, hv=32, lens=_text([1] * 64), fresh=False),
        # drafts of two to seven tokens of 24 sequences being verified
        dict(name="gdn_verify_b24", op="gdn", h=16, hv=32, lens=_text([2 + (5 * i) % 6 for i in range(24)]), fresh=False),
        # a batch of ragged prompts, continued from states (chunked prefill), four value heads a key head
        dict(name="gdn_ragged_b12", op="gdn", h=8, hv=32, lens="65,1531,64,700,1,2047,333,128,910,1279,17,256", fresh=False),
        # one long prompt from an empty state
        dict(name="gdn_prompt_8k", op="gdn", h=16, hv=32, lens="8192", fresh=True),
        # one token of two sequences through norm, rotation and append (latency)
        dict(name="append_b2", op="append", tokens=2, hq=16, hk=4, d=128, rot=128, inter=False, norm=True, page=16, pad=0),
        # a mixed step of 1001 tokens, some of them padding; interleaved rotation of the whole head, no norm
        dict(name="append_1k_inter", op="append", tokens=1001, hq=32, hk=8, d=128, rot=128, inter=True, norm=False, page=64, pad=23),
        # a prompt of 8192 tokens, wide heads, a quarter of each rotated
        dict(name="append_8k_partial", op="append", tokens=8192, hq=16, hk=2, d=256, rot=64, inter=False, norm=True, page=64, pad=0),
        # one sequence far into a long context, one new token
        dict(name="attn_token_50k", op="attn", q="1", kv="50001", hq=16, hk=2, d=128, page=16, lse=False),
        # 64 sequences generating, contexts of 100 to 8000 tokens
        dict(name="attn_token_b64", op="attn", q=_text([1] * 64), kv=_text(decode_ctx), hq=16, hk=4, d=128, page=64, lse=False),
        # a mixed step: generating sequences next to chunks of prompts; wide heads
        dict(name="attn_mixed", op="attn", q="1,1,1,1,5,300,1,1,701,1,1,33", kv="2000,17,4097,900,1205,300,64,1,2749,3333,511,4000", hq=16, hk=2, d=256,
             page=32, lse=True),
        # a chunk of 2048 tokens of a prompt that is already 30 k tokens long
        dict(name="attn_chunk_32k", op="attn", q="2048", kv="32768", hq=16, hk=2, d=128, page=64, lse=False),
    ]


def _loguniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _not(value, without=3072):
    return value + 1 if value == without else value


def draw(rng):
    op = rng.choice(["gdn", "append", "attn"])
    if op == "gdn":
        h, hv = rng.choice([(16, 32), (16, 16), (8, 32), (8, 16), (4, 8)])
        kind = rng.choice(["token", "short", "prompt"])
        if kind == "token":
            lens = [1] * _loguniform(rng, 1, 128)
        elif kind == "short":
            lens = [rng.randint(1, 12) for _ in range(_loguniform(rng, 1, 32))]
        else:
            n = _loguniform(rng, 1, 16)
            top = 8000 // n if n > 4 else 6000 // n
            lens = [_not(_loguniform(rng, 1, max(64, top))) for _ in range(n)]
        return dict(op=op, h=h, hv=hv, lens=_text(lens), fresh=rng.random() < 0.5)
    if op == "append":
        hq, hk = rng.choice([(16, 4), (16, 2), (32, 8), (8, 8), (14, 2)])
        d = rng.choice([64, 128, 256])
        tokens = _not(_loguniform(rng, 1, 8192 * 16 // max(16, hq)))
        return dict(op=op, tokens=tokens, hq=hq, hk=hk, d=d, rot=rng.choice([d, d // 2, d // 4]), inter=rng.random() < 0.5,
                    norm=rng.random() < 0.7, page=rng.choice([16, 24, 32, 64, 128]), pad=rng.randint(0, tokens // 8))
    hq, hk = rng.choice([(16, 4), (16, 2), (32, 8), (8, 8), (14, 2)])
    d = rng.choice([64, 128, 256])
    page = rng.choice([16, 24, 32, 64, 128])
    kind = rng.choice(["token", "chunk", "mixed"])
    if kind == "token":
        n = _loguniform(rng, 1, 96)
        q = [1] * n
        kv = [_not(_loguniform(rng, 1, min(32768, 400000 // n))) for _ in range(n)]
    elif kind == "chunk":
        n = rng.randint(1, 3)
        q = [_not(_loguniform(rng, 16, 2048 // n)) for _ in range(n)]
        kv = [_not(x + rng.choice([0, _loguniform(rng, 1, 16384 // n)])) for x in q]
    else:
        n = rng.randint(2, 16)
        q = [1 if rng.random() < 0.7 else _loguniform(rng, 2, 600) for _ in range(n)]
        kv = [_not(x + _loguniform(rng, 1, 4000)) for x in q]
    return dict(op=op, q=_text(q), kv=_text(kv), hq=hq, hk=hk, d=d, page=page, lse=rng.random() < 0.5)


# ----------------------------------------------------------------------------------------- inputs
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return {"gdn": _prepare_gdn, "append": _prepare_append, "attn": _prepare_attn}[case["op"]](case, g)


def _prepare_gdn(case, g):
    h, hv, lens = case["h"], case["hv"], _lens(case["lens"])
    n, total = len(lens), sum(lens)
    bf = torch.bfloat16
    # the repository's decode distributions: raw q|k|v and a, b ~ N(0,1), A = U(1,16), dt_bias ~ N(0, 0.5)
    s = {
        "op": "gdn", "h": h, "hv": hv, "lens": lens, "max_len": max(lens),
        "mixed": _randn(g, total, 2 * h * 128 + hv * 128).to(bf),
        "a": _randn(g, total, hv).to(bf), "b": _randn(g, total, hv).to(bf),
        "a_log": torch.log(1.0 + 15.0 * torch.rand(hv, generator=g, device=DEV)),
        "dt_bias": 0.5 * _randn(g, hv),
        # states a sequence arrives with; a fresh prompt's slot holds what its last user left
        "state": 0.05 * _randn(g, n, hv, 128, 128),
        "cu": torch.tensor([0] + lens, device=DEV).cumsum(0).to(torch.int32),
        "has_initial": torch.full((n,), not case["fresh"], dtype=torch.bool, device=DEV),
    }
    return s


def _rope_table(positions, rot):
    inv = 10000.0 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
    ang = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * inv
    return torch.cat([ang.cos(), ang.sin()], 1).float()


def _prepare_append(case, g):
    t, hq, hk, d, page = (case[k] for k in ("tokens", "hq", "hk", "d", "page"))
    pages = -(-t // page) + 3
    bf = torch.bfloat16
    order = torch.randperm(pages, generator=g, device=DEV)
    at = torch.arange(t, device=DEV)
    slots = order[at // page] * page + at % page
    if case["pad"]:
        slots[torch.randperm(t, generator=g, device=DEV)[:case["pad"]]] = -1  # padding rows are not appended
    qkv = _randn(g, t, (hq + 2 * hk) * d).to(bf)
    return {
        "op": "append", "hq": hq, "hk": hk, "d": d, "rot": case["rot"], "inter": case["inter"],
        "q": qkv[:, :hq * d].view(t, hq, d), "k": qkv[:, hq * d:(hq + hk) * d].view(t, hk, d), "v": qkv[:, (hq + hk) * d:].view(t, hk, d),
        "qw": (1.0 + 0.2 * _randn(g, d)).to(bf) if case["norm"] else None,
        "kw": (1.0 + 0.2 * _randn(g, d)).to(bf) if case["norm"] else None,
        "positions": (torch.randint(0, 20000, (1,), generator=g, device=DEV) + at).to(torch.int32),
        "slots": slots.to(torch.int32),
        "table": _rope_table(20000 + t, case["rot"]),
        "k_cache": _randn(g, pages, page, hk, d).to(bf), "v_cache": _randn(g, pages, page, hk, d).to(bf),
    }


def _prepare_attn(case, g):
    q, kv, hq, hk, d, page = _lens(case["q"]), _lens(case["kv"]), case["hq"], case["hk"], case["d"], case["page"]
    used = [-(-x // page) for x in kv]
    pages, widest = sum(used) + 2, max(used)
    bf = torch.bfloat16
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    begin = torch.tensor([0] + used, device=DEV).cumsum(0)[:-1]
    at = torch.arange(widest, device=DEV)[None, :]
    table = order[(begin[:, None] + at).clamp(max=pages - 1)]
    table = torch.where(at < torch.tensor(used, device=DEV)[:, None], table, torch.zeros_like(table))
    return {
        "op": "attn", "hq": hq, "hk": hk, "d": d, "page": page, "q_lens": q, "kv_list": kv, "max_q": max(q), "lse": case["lse"],
        "q": (1.5 * _randn(g, sum(q), hq, d)).to(bf),
        "k_cache": _randn(g, pages, page, hk, d).to(bf), "v_cache": _randn(g, pages, page, hk, d).to(bf),
        "table": table.contiguous(), "kv_lens": torch.tensor(kv, dtype=torch.int32, device=DEV),
        "cu": torch.tensor([0] + q, device=DEV).cumsum(0).to(torch.int32),
    }


# -------------------------------------------------------------------------------------------- run
def run(state):
    return {"gdn": _run_gdn, "append": _run_append, "attn": _run_attn}[state["op"]](state)


def _run_gdn(s):
    if own:
        out = _package().gdn_prefill(s["mixed"], s["a"], s["b"], s["a_log"], s["dt_bias"], s["state"], s["cu"],
                                     has_initial_state=s["has_initial"], max_seqlen=s["max_len"])
        return {"out": out, "state": s["state"]}
    out, final = _plain_gdn(s)
    s["state"].copy_(final)
    return {"out": out, "state": s["state"]}


def _pad_index(cu, n, width):
    """[N, width] token index of each padded place, and whether it is a token."""
    at = torch.arange(width, device=DEV)[None, :]
    lens = (cu[1:] - cu[:-1]).long()[:, None]
    valid = at < lens
    return torch.where(valid, cu[:-1].long()[:, None] + at, torch.zeros_like(at)), valid


def _plain_gdn(s):
    """Chunks of up to 64 tokens of the padded batch: what does not need the state for all chunks at once, then a loop
    that carries the state over the chunks."""
    h, hv, n = s["h"], s["hv"], len(s["lens"])
    c = min(64, s["max_len"])
    chunks = -(-s["max_len"] // c)
    at, valid = _pad_index(s["cu"], n, chunks * c)
    x = s["mixed"].float()[at] * valid[..., None]  # [N, T, W]

    def heads(y, k):  # [N, T, k*128] -> [N, HV, chunks, C, 128]
        y = y.view(n, chunks, c, k, 128).permute(0, 3, 1, 2, 4)
        return y.repeat_interleave(hv // k, 1)

    q, k, v = heads(x[..., :h * 128], h), heads(x[..., h * 128:2 * h * 128], h), heads(x[..., 2 * h * 128:], hv)
    q = q * torch.rsqrt((q * q).sum(-1, keepdim=True) + EPS) * 128 ** -0.5
    k = k * torch.rsqrt((k * k).sum(-1, keepdim=True) + EPS)
    t = s["a"].float()[at] + s["dt_bias"]
    gate = -torch.exp(s["a_log"]) * torch.where(t > 20, t, torch.log1p(torch.exp(t.clamp(max=20))))
    gate = (gate * valid[..., None]).view(n, chunks, c, hv).permute(0, 3, 1, 2)  # padding neither decays nor writes
    beta = (torch.sigmoid(s["b"].float()[at]) * valid[..., None]).view(n, chunks, c, hv).permute(0, 3, 1, 2)
    low = torch.ones(c, c, device=DEV, dtype=torch.bool).tril(-1)
    # sum of the gates of tokens j+1 .. i, summed as such: differences of prefix sums would cancel under strong decay
    span = (gate[..., :, None] * low).cumsum(-2)
    decay = torch.exp(span) * (low | torch.eye(c, device=DEV, dtype=torch.bool))
    prefix = torch.exp(gate.cumsum(-1))[..., None]  # from the chunk's start
    suffix = decay[..., -1, :, None]  # to the chunk's end
    m = -(beta[..., None] * (k @ k.mT) * decay * low)
    inv = torch.eye(c, device=DEV) + m  # (I - m)^-1 = (I + m)(I + m^2)(I + m^4)...: m is nilpotent
    p, power = m, 2
    while power < c:
        p = p @ p
        inv = inv + inv @ p
        power *= 2
    scores = (q @ k.mT) * decay
    fixed = inv @ (beta[..., None] * v)
    seen = inv @ (beta[..., None] * prefix * k)
    state = s["state"] * s["has_initial"][:, None, None, None]
    outs = []
    for i in range(chunks):
        new = fixed[:, :, i] - seen[:, :, i] @ state.mT
        outs.append(prefix[:, :, i] * (q[:, :, i] @ state.mT) + scores[:, :, i] @ new)
        state = prefix[:, :, i, -1:] * state + (new * suffix[:, :, i]).mT @ k[:, :, i]
    out = torch.stack(outs, 2).permute(0, 2, 3, 1, 4).reshape(n, chunks * c, hv, 128)
    return out[valid].to(torch.bfloat16), state


def _rotate(x, cos, sin, rot, inter):
    r = x[..., :rot]
    x1, x2 = (r[..., 0::2], r[..., 1::2]) if inter else (r[..., :rot // 2], r[..., rot // 2:])
    y1, y2 = x1 * cos - x2 * sin, x2 * cos + x1 * sin
    y = torch.stack([y1, y2], -1).flatten(-2) if inter else torch.cat([y1, y2], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _norm_rotate(s, x, weight, dtype):
    x = x.to(dtype)
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.to(dtype)
    row = s["table"][s["positions"].long()].to(dtype)[:, None, :]
    return _rotate(x, row[..., :s["rot"] // 2], row[..., s["rot"] // 2:], s["rot"], s["inter"])


def _run_append(s):
    if own:
        q = _package().qk_norm_rope_append(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["table"], s["k_cache"], s["v_cache"],
                                           q_weight=s["qw"], k_weight=s["kw"], eps=EPS, interleaved=s["inter"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    q = _norm_rotate(s, s["q"], s["qw"], torch.float32).to(torch.bfloat16)
    k = _norm_rotate(s, s["k"], s["kw"], torch.float32).to(torch.bfloat16)
    keep = s["slots"] >= 0
    to = s["slots"][keep].long()
    s["k_cache"].view(-1, s["hk"], s["d"])[to] = k[keep]
    s["v_cache"].view(-1, s["hk"], s["d"])[to] = s["v"][keep]
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _run_attn(s):
    if own:
        if s["lse"]:
            out, lse = _package().paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["kv_lens"], s["cu"],
                                                  max_seqlen=s["max_q"], return_lse=True)
            return {"out": out, "lse": lse}
        return {"out": _package().paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["kv_lens"], s["cu"], max_seqlen=s["max_q"])}
    n, hq, hk, d, m = len(s["q_lens"]), s["hq"], s["hk"], s["d"], s["max_q"]
    at, valid = _pad_index(s["cu"], n, m)
    width = s["table"].shape[1] * s["page"]
    q = s["q"].float()[at].view(n, m, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(n, hk, hq // hk * m, d)
    k = s["k_cache"][s["table"].long()].float().view(n, width, hk, d).permute(0, 2, 1, 3)
    v = s["v_cache"][s["table"].long()].float().view(n, width, hk, d).permute(0, 2, 1, 3)
    kv = s["kv_lens"].long()
    # the new tokens are the last of the sequence: row i of m_n sees places up to kv_n - m_n + i
    last = (kv - (s["cu"][1:] - s["cu"][:-1]).long())[:, None] + torch.arange(m, device=DEV)
    see = (torch.arange(width, device=DEV) <= last[..., None]) & valid[..., None]  # [N, M, width]
    scores = ((q * d ** -0.5) @ k.mT).view(n, hk, hq // hk, m, width)
    scores = scores.masked_fill_(~see[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores.sub_(torch.where(torch.isfinite(top), top, torch.zeros_like(top))))
    total = p.sum(-1, keepdim=True)
    out = (p.view(n, hk, -1, width) @ v).view(n, hk, hq // hk, m, d) / torch.where(total > 0, total, torch.ones_like(total))
    out = out.permute(0, 3, 1, 2, 4).reshape(n, m, hq, d)[valid].to(torch.bfloat16)
    if not s["lse"]:
        return {"out": out}
    lse = (torch.log(total) + top).squeeze(-1).permute(0, 3, 1, 2).reshape(n, m, hq)[valid]
    return {"out": out, "lse": lse}


# ------------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "gdn":
        lens, h, hv = _lens(case["lens"]), case["h"], case["hv"]
        t, n = sum(lens), len(lens)
        states = n * hv * 128 * 128 * 4
        moved = t * (2 * h * 128 + hv * 128) * 2 + t * hv * 2 * 2 + t * hv * 128 * 2 + states * (1 if case["fresh"] else 2)
        # a token of a head: S k, the decayed rank-one update, S q
        return {"bytes": moved, "flops": 6.0 * 128 * 128 * hv * t}
    if case["op"] == "append":
        t, hq, hk, d = case["tokens"], case["hq"], case["hk"], case["d"]
        return {"bytes": 2 * t * (hq + 2 * hk) * d * 2 + t * (case["rot"] * 4 + 8), "flops": t * (hq + hk) * (4 * d + 3 * case["rot"])}
    q, kv, hq, hk, d = _lens(case["q"]), _lens(case["kv"]), case["hq"], case["hk"], case["d"]
    seen = sum(sum(max(0, y - x + 1 + i) for i in range(x)) for x, y in zip(q, kv))
    moved = sum(q) * hq * d * 2 * 2 + sum(kv) * hk * d * 2 * 2 + sum(-(-y // case["page"]) for y in kv) * 4
    return {"bytes": moved + (sum(q) * hq * 4 if case["lse"] else 0), "flops": 4.0 * d * hq * seen}


# ------------------------------------------------------------------------------------------ exact
def exact(case, seed):
    s = prepare(case, seed)
    return {"gdn": _exact_gdn, "append": _exact_append, "attn": _exact_attn}[case["op"]](s)


def _exact_gdn(s):
    """The recurrence itself, token by token, in float64: the sequences side by side, longest first."""
    h, hv, lens = s["h"], s["hv"], s["lens"]
    f = torch.float64
    x = s["mixed"].to(f)
    q, k, v = x[:, :h * 128].view(-1, h, 128), x[:, h * 128:2 * h * 128].view(-1, h, 128), x[:, 2 * h * 128:].view(-1, hv, 128)
    q = (q / torch.sqrt((q * q).sum(-1, keepdim=True) + EPS) * 128 ** -0.5).repeat_interleave(hv // h, 1)
    k = (k / torch.sqrt((k * k).sum(-1, keepdim=True) + EPS)).repeat_interleave(hv // h, 1)
    t = s["a"].to(f) + s["dt_bias"].to(f)
    alpha = torch.exp(-torch.exp(s["a_log"].to(f)) * torch.log1p(torch.exp(t)))
    beta = 1.0 / (1.0 + torch.exp(-s["b"].to(f)))
    order = sorted(range(len(lens)), key=lambda i: -lens[i])
    first = s["cu"].long()[:-1][torch.tensor(order, device=DEV)]
    state = (s["state"].to(f) * s["has_initial"][:, None, None, None])[torch.tensor(order, device=DEV)].contiguous()
    out = torch.zeros(len(x), hv, 128, dtype=f, device=DEV)
    live = len(lens)
    for i in range(max(lens)):
        while live and lens[order[live - 1]] <= i:
            live -= 1
        at = first[:live] + i
        st, ki = state[:live], k[at][:, :, :, None]
        st.mul_(alpha[at][:, :, None, None])
        delta = beta[at][:, :, None] * (v[at] - (st @ ki)[..., 0])
        st.add_(delta[..., None] * ki.mT)
        out[at] = (st @ q[at][..., None])[..., 0]
    final = torch.empty_like(state)
    final[torch.tensor(order, device=DEV)] = state
    return {"out": out, "state": final}


def _exact_append(s):
    f = torch.float64
    q, k = _norm_rotate64(s, s["q"], s["qw"]), _norm_rotate64(s, s["k"], s["kw"])
    kc, vc = s["k_cache"].to(f), s["v_cache"].to(f)
    keep = (s["slots"] >= 0).nonzero()[:, 0]
    page = kc.shape[1]
    to = s["slots"].long()[keep]
    kc[to // page, to % page] = k[keep]
    vc[to // page, to % page] = s["v"].to(f)[keep]
    return {"q": q, "k_cache": kc, "v_cache": vc}


def _norm_rotate64(s, x, weight):
    """As a product of complex numbers."""
    x = x.to(torch.float64)
    if weight is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * weight.to(torch.float64)
    half = s["rot"] // 2
    turn = s["table"].to(torch.float64)[s["positions"].long()]
    turn = torch.complex(turn[:, :half], turn[:, half:])[:, None, :]
    first = torch.arange(half, device=DEV) * 2 if s["inter"] else torch.arange(half, device=DEV)
    second = first + 1 if s["inter"] else first + half
    z = torch.complex(x[..., first], x[..., second]) * turn
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_attn(s):
    f = torch.float64
    outs, lses = [], []
    group = s["hq"] // s["hk"]
    cu = s["cu"].tolist()
    for i, (m, n) in enumerate(zip(s["q_lens"], s["kv_list"])):
        pages = s["table"][i, :-(-n // s["page"])].long()
        k = s["k_cache"][pages].flatten(0, 1)[:n].to(f)
        v = s["v_cache"][pages].flatten(0, 1)[:n].to(f)
        hidden = torch.arange(n, device=DEV)[None, :] > torch.arange(n - m, n, device=DEV)[:, None]
        per, low = [], []
        for head in range(s["hq"]):
            x = s["q"][cu[i]:cu[i + 1], head].to(f) @ k[:, head // group].T / math.sqrt(s["d"])
            x.masked_fill_(hidden, -math.inf)
            l = torch.logsumexp(x, -1, keepdim=True)
            per.append(torch.exp(x - l) @ v[:, head // group])
            low.append(l[:, 0])
        outs.append(torch.stack(per, 1))
        lses.append(torch.stack(low, 1))
    out = torch.cat(outs)
    return {"out": out, "lse": torch.cat(lses)} if s["lse"] else {"out": out}
