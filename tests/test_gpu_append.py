"""qk_norm_rope_append against its formulas in float64.

A stored value is rounded once to bf16: half a unit in the last place is at most 2^-8 of the
value, and float32 arithmetic before it adds far less than 1e-5 of the row's largest value.
"""

import pytest
import torch

import gdnr
import hybrid_ref as R

pytestmark = pytest.mark.gpu


def near(got, want):
    top = want.abs().amax(-1, keepdim=True)
    assert ((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5 * top + 1e-30).all()


def make(seed, t, hq, hk, d, page, pages, rot):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def n(*s):
        return torch.randn(*s, generator=g, device="cuda")

    qkv = n(t, (hq + 2 * hk) * d).bfloat16()
    return dict(q=qkv[:, :hq * d].view(t, hq, d), k=qkv[:, hq * d:(hq + hk) * d].view(t, hk, d), v=qkv[:, (hq + hk) * d:].view(t, hk, d),
                positions=torch.randint(0, 1000, (t,), generator=g, device="cuda").int(),
                slots=torch.randperm(page * pages, generator=g, device="cuda")[:t].int(),
                table=gdnr.rope_table(1000, rot) if rot else torch.empty(1000, 0, device="cuda"),
                kc=n(pages, page, hk, d).bfloat16(), vc=n(pages, page, hk, d).bfloat16(),
                qw=(1 + 0.3 * n(d)).bfloat16(), kw=1 + 0.3 * n(d))


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("t,hq,hk,d,page,rot,norm,offset", [
    (1, 4, 1, 64, 16, 64, True, 0.0),
    (5, 3, 3, 128, 7, 10, True, 1.0),
    (33, 8, 2, 256, 32, 64, True, 0.0),
    (9, 1, 1, 256, 1, 250, True, 0.0),
    (130, 14, 2, 64, 24, 32, False, 0.0),
    (17, 4, 4, 128, 16, 128, False, 0.0),
    (12, 2, 1, 128, 16, 2, True, 0.0),
    (6, 2, 1, 64, 16, 0, True, 0.0),
])
def test_against_formulas(cuda_device, t, hq, hk, d, page, rot, norm, offset, inter):
    x = make(t * d + rot, t, hq, hk, d, page, -(-t // page) + 2, rot)
    x["slots"][::4] = -1
    if t == 1:
        x["slots"][:] = 17
    qw, kw = (x["qw"], x["kw"]) if norm else (None, None)
    kc, vc = x["kc"].clone(), x["vc"].clone()
    gdnr.read_device_error()
    q = gdnr.qk_norm_rope_append(x["q"], x["k"], x["v"], x["positions"], x["slots"], x["table"], kc, vc, q_weight=qw, k_weight=kw,
                                 weight_offset=offset, eps=1e-5, interleaved=inter)
    assert gdnr.read_device_error() == 0
    rows = x["table"][x["positions"].long()]
    near(q, R.norm_rope(x["q"], qw, offset, 1e-5, rows, inter))
    k = R.norm_rope(x["k"], kw, offset, 1e-5, rows, inter)
    keep = x["slots"] >= 0
    to = x["slots"][keep].long()
    near(kc.view(-1, hk, d)[to], k[keep])
    assert torch.equal(vc.view(-1, hk, d)[to], x["v"][keep])
    rest = torch.ones(kc.shape[0] * page, dtype=torch.bool, device="cuda")
    rest[to] = False
    assert torch.equal(kc.view(-1, hk, d)[rest], x["kc"].view(-1, hk, d)[rest])
    assert torch.equal(vc.view(-1, hk, d)[rest], x["vc"].view(-1, hk, d)[rest])


def test_only_queries_normed_and_in_place(cuda_device):
    x = make(1, 20, 4, 2, 128, 16, 3, 128)
    q = x["q"].clone()
    k0 = R.norm_rope(x["k"], None, 0, 0, x["table"][x["positions"].long()], False)
    want = R.norm_rope(q, x["qw"], 0, 1e-6, x["table"][x["positions"].long()], False)
    got = gdnr.qk_norm_rope_append(q, x["k"], x["v"], x["positions"], x["slots"], x["table"], x["kc"], x["vc"], q_weight=x["qw"], q_out=q)
    assert got.data_ptr() == q.data_ptr()
    near(q, want)
    near(x["kc"].view(-1, 2, 128)[x["slots"].long()], k0)


def test_strided_caches_and_inputs(cuda_device):
    """K and V interleaved in one buffer, [pages, 2, Hk, page, D] with the head before the row."""
    t, hk, d, page, pages = 21, 2, 64, 8, 5
    x = make(2, t, 4, hk, d, page, pages, 64)
    buf = torch.zeros(pages, 2, hk, page, d, dtype=torch.bfloat16, device="cuda")
    kc, vc = buf[:, 0].transpose(1, 2), buf[:, 1].transpose(1, 2)
    pos = torch.stack([x["positions"]] * 2, 1)[:, 0]
    gdnr.qk_norm_rope_append(x["q"], x["k"], x["v"], pos, x["slots"], x["table"], kc, vc, k_weight=x["kw"])
    s = x["slots"].long()
    near(kc[s // page, s % page], R.norm_rope(x["k"], x["kw"], 0, 1e-6, x["table"][x["positions"].long()], False))
    assert torch.equal(vc[s // page, s % page], x["v"])


def test_bad_slot_and_position_are_reported(cuda_device):
    x = make(3, 8, 2, 1, 64, 4, 3, 64)
    x["slots"][2] = 12  # one past the cache
    kc, vc = x["kc"].clone(), x["vc"].clone()
    gdnr.read_device_error()
    gdnr.qk_norm_rope_append(x["q"], x["k"], x["v"], x["positions"], x["slots"], x["table"], kc, vc)
    assert gdnr.read_device_error() == 0x8
    x["slots"][2] = -1
    x["positions"][1], x["positions"][5] = 1000, -1
    q = gdnr.qk_norm_rope_append(x["q"], x["k"], x["v"], x["positions"], x["slots"], x["table"], kc, vc)
    assert gdnr.read_device_error() == 0x2
    assert torch.equal(q[1], x["q"][1]) and torch.equal(q[5], x["q"][5])


def test_infinities_and_nan_stay_in_their_head(cuda_device):
    x = make(4, 6, 4, 2, 128, 16, 2, 64)
    x["q"][1, 2, 5] = float("nan")
    x["k"][3, 1, 100] = float("inf")
    q = gdnr.qk_norm_rope_append(x["q"], x["k"], x["v"], x["positions"], x["slots"], x["table"], x["kc"], x["vc"], q_weight=x["qw"], k_weight=x["kw"])
    bad = torch.zeros(6, 4, dtype=torch.bool, device="cuda")
    bad[1, 2] = True
    assert torch.equal(torch.isnan(q).any(-1), bad)
    k = x["kc"].view(-1, 2, 128)[x["slots"].long()]
    assert torch.isnan(k[3, 1]).any() and torch.isfinite(k[3, 0]).all() and torch.isfinite(k[:3]).all() and torch.isfinite(k[4:]).all()


def test_no_tokens(cuda_device):
    x = make(5, 4, 2, 1, 64, 4, 2, 64)
    q = gdnr.qk_norm_rope_append(x["q"][:0], x["k"][:0], x["v"][:0], x["positions"][:0], x["slots"][:0], x["table"], x["kc"], x["vc"])
    assert q.shape == (0, 2, 64)


def test_cache_offsets_past_32_bits(cuda_device):
    hk, d, page = 8, 128, 64
    pages = 2 ** 32 // (hk * d * page) + 2
    x = make(6, 3, 8, hk, d, page, 1, 128)
    kc, vc = (torch.empty(pages, page, hk, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    slots = torch.tensor([pages * page - 1, 0, (pages - 1) * page], dtype=torch.int32, device="cuda")
    gdnr.qk_norm_rope_append(x["q"], x["k"], x["v"], x["positions"], slots, x["table"], kc, vc)
    k = R.norm_rope(x["k"], None, 0, 0, x["table"][x["positions"].long()], False)
    near(torch.stack([kc[-1, -1], kc[0, 0], kc[-1, 0]]), k)
    assert torch.equal(torch.stack([vc[-1, -1], vc[0, 0], vc[-1, 0]]), x["v"])


def test_rope_table_scaling():
    """linear: positions divided; yarn: fast pairs keep, slow pairs are divided, gain 0.1 ln(factor) + 1."""
    plain, lin = gdnr.rope_table(64, 32, device="cpu"), gdnr.rope_table(64, 32, scaling="linear", factor=4.0, device="cpu")
    assert torch.allclose(lin[::4], plain[:16], atol=1e-6)
    yarn = gdnr.rope_table(64, 64, scaling="yarn", factor=8.0, original_positions=4096, device="cpu")
    gain = 0.1 * torch.log(torch.tensor(8.0)) + 1
    wide = gdnr.rope_table(64, 64, device="cpu")
    assert torch.allclose(yarn[:, 0], gain * wide[:, 0], atol=1e-5)  # turns 4096 / 2 pi times: kept
    slow = torch.cos(torch.arange(64) * 10000.0 ** (-62 / 64) / 8)
    assert torch.allclose(yarn[:, 31], gain * slow, atol=1e-5)
    for bad in (dict(rot_dim=7), dict(rot_dim=8, scaling="other"), dict(rot_dim=8, scaling="yarn", factor=2.0), dict(rot_dim=8, factor=0.5)):
        with pytest.raises(ValueError):
            gdnr.rope_table(4, device="cpu", **bad)
