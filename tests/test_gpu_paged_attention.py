"""paged_attention against softmax attention in float64.

Tolerances: out (relative 2-norm) 5e-3 -- rounding to bf16 is 1.7e-3 rms, of the weights and of the
stored value, 2.4e-3 together, twice that allowed.  lse: float32 dot products of D <= 256
terms of size about one, scaled by D^-1/2: 3e-5 absolute.
"""

import math

import pytest
import torch

import gdnr
import hybrid_ref as R

pytestmark = pytest.mark.gpu

TOL_OUT, TOL_LSE = 5e-3, 3e-5


def make(seed, q_lens, kv_lens, hq, hk, d, page, spare=2):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    used = [-(-k // page) for k in kv_lens]
    pages = sum(used) + spare

    def n(*s):
        return torch.randn(*s, generator=g, device="cuda").bfloat16()

    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((len(q_lens), max(max(used, default=1), 1)), -1, dtype=torch.int32, device="cuda")  # never read past the end
    at = 0
    for i, u in enumerate(used):
        table[i, :u] = order[at:at + u]
        at += u
    return dict(q=n(sum(q_lens), hq, d), kc=n(pages, page, hk, d), vc=n(pages, page, hk, d), table=table,
                kv=torch.tensor(kv_lens, dtype=torch.int32, device="cuda"), q_lens=q_lens)


def check(x, scale=None, hint=None, **kw):
    d = x["q"].shape[-1]
    gdnr.read_device_error()
    out, lse = gdnr.paged_attention(x["q"], x["kc"], x["vc"], x["table"], x["kv"], R.cu(x["q_lens"]), scale=scale, return_lse=True,
                                    max_seqlen=max(x["q_lens"], default=0) if hint is None else hint, **kw)
    assert gdnr.read_device_error() == 0
    want, low = R.attention(x["q"], x["kc"], x["vc"], x["table"], x["kv"], x["q_lens"], d ** -0.5 if scale is None else scale)
    assert torch.isfinite(out).all()
    empty = torch.isinf(low)
    assert torch.equal(torch.isinf(lse) & (lse < 0), empty)
    assert (out[empty] == 0).all()
    if (~empty).any():
        assert R.rel(out[~empty], want[~empty]) < TOL_OUT
        assert float((lse.double() - low)[~empty].abs().max()) < TOL_LSE
        # and row by row, so that one wrong row of many is seen: four times the whole's tolerance
        err = (out.double() - want)[~empty].norm(dim=-1) / want[~empty].norm(dim=-1).clamp(min=1e-6)
        assert float(err.max()) < 4 * TOL_OUT
    return out, lse


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hk", [(8, 1), (4, 4), (14, 2), (32, 2)])
@pytest.mark.parametrize("page", [1, 16, 24, 64, 128])
def test_single_tokens(cuda_device, d, hq, hk, page):
    check(make(d + hq + page, [1, 1, 1, 1, 1], [1, 63, 64, 65, 700], hq, hk, d, page))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hk", [(8, 1), (4, 4), (14, 2)])
@pytest.mark.parametrize("page", [5, 16, 64, 256])
def test_chunks_and_single_tokens_together(cuda_device, d, hq, hk, page):
    check(make(d + hq + page, [1, 40, 3, 130, 1, 257], [500, 40, 129, 400, 1, 300], hq, hk, d, page))


@pytest.mark.parametrize("q_lens,kv_lens", [([64], [64]), ([63], [190]), ([128], [128]), ([127], [129]), ([1], [4000]), ([300], [2100]), ([513], [513])])
def test_tile_edges(cuda_device, q_lens, kv_lens):
    for d in (128, 256):
        check(make(sum(kv_lens), q_lens, kv_lens, 8, 2, d, 32))


@pytest.mark.parametrize("hq,hk", [(40, 1), (24, 1), (64, 1), (5, 1), (130, 1)])
def test_many_query_heads_for_one_key_head(cuda_device, hq, hk):
    check(make(hq, [1, 2, 60], [100, 70, 333], hq, hk, 128, 16))


def test_rows_without_places(cuda_device):
    """Sequences whose cache is shorter than their new tokens, or empty; empty sequences."""
    for q_lens, kv_lens in (([4, 1, 0, 3, 2], [2, 0, 5, 0, 2]), ([200, 1, 0, 150], [150, 9, 70, 0]), ([0, 0], [3, 0])):
        check(make(1, q_lens, kv_lens, 8, 2, 128, 16))


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [70, 130]), ([100, 300], [190, 333])])
@pytest.mark.parametrize("fill", [float("nan"), float("inf"), 3.3e38])
def test_garbage_past_the_end_is_not_used(cuda_device, q_lens, kv_lens, fill):
    """What freed pages and the rest of the last page hold."""
    for d, page in ((128, 16), (128, 24), (256, 64)):
        x = make(2, q_lens, kv_lens, 8, 2, d, page)
        clean, _ = check(x)
        free = torch.ones(x["kc"].shape[:2], dtype=torch.bool, device="cuda")
        for i, kv in enumerate(kv_lens):
            at = torch.arange(kv, device="cuda")
            free[x["table"][i, at // page].long(), at % page] = False
        x["kc"][free], x["vc"][free] = fill, fill
        out, _ = check(x)
        assert torch.equal(out, clean)


def test_scores_of_any_size(cuda_device):
    """Scores of hundreds (one key takes all) and scores that are all equal."""
    for lens in ([1, 3], [150, 70]):
        x = make(3, lens, [400, 333], 8, 2, 128, 16)
        x["q"] *= 40
        gdnr.read_device_error()
        out = gdnr.paged_attention(x["q"], x["kc"], x["vc"], x["table"], x["kv"], R.cu(lens), max_seqlen=max(lens))
        want, _ = R.attention(x["q"], x["kc"], x["vc"], x["table"], x["kv"], lens, 128 ** -0.5)
        assert R.rel(out, want) < 2 * TOL_OUT  # scores of 500 in float32: 3e-5 of a weight's exponent, still far below
        x["q"].zero_()
        check(x)


@pytest.mark.parametrize("scale", [0.0, 0.01, -0.2])
def test_scale(cuda_device, scale):
    check(make(4, [1, 20], [90, 200], 4, 2, 64, 16), scale=scale)


def test_strided_tensors(cuda_device):
    """[pages, 2, Hk, page, D] buffer, queries out of a wider projection, a wider out, every second table row."""
    q_lens, kv_lens, hk, d, page = [1, 150, 7], [33, 150, 220], 2, 128, 32
    x = make(5, q_lens, kv_lens, 8, hk, d, page)
    buf = torch.empty(x["kc"].shape[0], 2, hk, page, d, dtype=torch.bfloat16, device="cuda")
    buf[:, 0], buf[:, 1] = x["kc"].transpose(1, 2), x["vc"].transpose(1, 2)
    x["kc"], x["vc"] = buf[:, 0].transpose(1, 2), buf[:, 1].transpose(1, 2)
    wide = torch.zeros(sum(q_lens), 12, d, dtype=torch.bfloat16, device="cuda")
    wide[:, 2:10] = x["q"]
    x["q"] = wide[:, 2:10]
    x["table"] = torch.stack([x["table"], x["table"] * 0 - 7], 1).flatten(0, 1)[::2]
    out = torch.full((sum(q_lens), 8, d + 8), float("nan"), dtype=torch.bfloat16, device="cuda")
    check(x, out=out[..., :d])
    assert torch.isnan(out[..., d:]).all()


def test_hint_unknown_or_large(cuda_device):
    x = make(6, [1, 2, 1], [100, 200, 3000], 8, 2, 128, 16)
    for hint in (0, 2, 5000):
        check(x, hint=hint)


def test_shared_pages(cuda_device):
    """Two sequences with the same prefix pages."""
    x = make(7, [1, 90], [256, 256], 8, 2, 128, 64)
    x["table"][1, :3] = x["table"][0, :3]
    check(x)


def test_page_outside_the_cache_is_reported(cuda_device):
    for lens in ([1], [200]):
        x = make(8, lens, [300], 8, 2, 128, 16)
        x["table"][0, 5] = x["kc"].shape[0]
        gdnr.read_device_error()
        out = gdnr.paged_attention(x["q"], x["kc"], x["vc"], x["table"], x["kv"], R.cu(lens), max_seqlen=lens[0])
        assert gdnr.read_device_error() & 0x8
        assert torch.isfinite(out).all()


def test_cache_offsets_past_32_bits(cuda_device):
    hk, d, page = 8, 128, 64
    pages = 2 ** 32 // (hk * d * page) + 3
    kc, vc = (torch.empty(pages, page, hk, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    for lens in ([1, 1], [150, 60]):
        x = make(9, lens, [190, 100], 16, hk, d, page, spare=0)
        high = pages - 1 - x["table"]
        for i in range(2):
            for j in range(x["table"].shape[1]):
                if x["table"][i, j] >= 0:
                    kc[high[i, j].item()], vc[high[i, j].item()] = x["kc"][x["table"][i, j].item()], x["vc"][x["table"][i, j].item()]
        small, _ = check(x)
        out = gdnr.paged_attention(x["q"], kc, vc, high.clamp(max=pages - 1).int().contiguous(), x["kv"], R.cu(lens), max_seqlen=max(lens))
        assert torch.equal(out, small)


def test_runs_are_equal_and_streams_independent(cuda_device):
    for lens in ([1] * 6, [1, 200, 1, 64, 3, 90]):
        x = make(10, lens, [2000, 200, 17, 900, 1205, 300], 16, 2, 128, 16)
        want, _ = check(x)
        c = R.cu(lens)
        streams = [torch.cuda.Stream() for _ in range(3)]
        outs = []
        torch.cuda.synchronize()
        for _ in range(4):
            for s in streams:
                with torch.cuda.stream(s):
                    outs.append(gdnr.paged_attention(x["q"], x["kc"], x["vc"], x["table"], x["kv"], c, max_seqlen=max(lens)))
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o, want)


def test_lse_joins_two_halves_of_a_context(cuda_device):
    """What lse is for: attention over two disjoint parts of a context, joined by their lse."""
    x = make(11, [1], [640], 8, 2, 128, 64)
    whole, _ = check(x)
    parts = [gdnr.paged_attention(x["q"], x["kc"], x["vc"], x["table"][:, s].contiguous(), torch.tensor([n], dtype=torch.int32, device="cuda"),
                                  R.cu([1]), max_seqlen=1, return_lse=True) for s, n in ((slice(0, 4), 256), (slice(4, 10), 384))]
    (o1, l1), (o2, l2) = parts
    l = torch.logaddexp(l1, l2)
    joined = o1.float() * (l1 - l).exp()[..., None] + o2.float() * (l2 - l).exp()[..., None]
    assert R.rel(joined, whole) < 2 * TOL_OUT
    assert math.isfinite(float(l.sum()))


@pytest.mark.parametrize("n", [33, 200])
def test_many_sequences(cuda_device, n):
    """More sequences than a warp has lanes, single tokens and a few chunks."""
    q_lens = [1] * n
    check(make(n, q_lens, [(37 * i) % 150 for i in range(n)], 8, 2, 64, 16))
    q_lens[5], q_lens[n - 1] = 70, 30
    check(make(n, q_lens, [70 + (37 * i) % 150 for i in range(n)], 8, 2, 128, 16))
