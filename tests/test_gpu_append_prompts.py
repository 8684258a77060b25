"""qk_norm_rope_append on batches that fill the machine: two sets of heads and several tokens a warp (from 4.9 MB of values on;
test_gpu_append.py has smaller ones).  Inputs, formulas and the tolerance are that file's.
"""

import pytest
import torch

import gdnr
import hybrid_ref as R
from test_gpu_append import make, near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("t,hq,hk,d,page,rot,norm,offset", [
    (1001, 32, 8, 128, 64, 128, False, 0.0),  # 2 tokens a warp, the last one alone
    (8192, 16, 2, 256, 64, 64, True, 0.0),  # 4
    (8191, 16, 2, 256, 64, 64, True, 1.0),  # 4, the last walk has 3
    (5003, 3, 1, 256, 24, 250, True, 0.0),  # heads that leave half a set; pairs anywhere in the head
    (4099, 14, 2, 64, 16, 32, True, 0.0),  # sets of eight heads, three quarters and a quarter of them there
    (6001, 9, 3, 64, 7, 10, True, 0.0),
    (3001, 5, 5, 128, 16, 0, True, 0.0),  # no rotation
])
def test_against_formulas(cuda_device, t, hq, hk, d, page, rot, norm, offset, inter):
    x = make(t + rot, t, hq, hk, d, page, -(-t // page) + 2, rot)
    g = torch.Generator(device="cuda")
    g.manual_seed(t)
    padding = torch.rand(t, generator=g, device="cuda") < 0.2
    padding[:7] = torch.tensor([True, False, True, True, True, True, False], device="cuda")
    padding[-1] = True
    x["slots"][padding] = -1
    qw, kw = (x["qw"], x["kw"]) if norm else (None, None)
    kc, vc = x["kc"].clone(), x["vc"].clone()
    gdnr.read_device_error()
    q = gdnr.qk_norm_rope_append(x["q"], x["k"], x["v"], x["positions"], x["slots"], x["table"], kc, vc, q_weight=qw, k_weight=kw,
                                 weight_offset=offset, eps=1e-5, interleaved=inter)
    assert gdnr.read_device_error() == 0
    rows = x["table"][x["positions"].long()]
    near(q, R.norm_rope(x["q"], qw, offset, 1e-5, rows, inter))
    k = R.norm_rope(x["k"], kw, offset, 1e-5, rows, inter)
    to = x["slots"][~padding].long()
    near(kc.view(-1, hk, d)[to], k[~padding])
    assert torch.equal(vc.view(-1, hk, d)[to], x["v"][~padding])
    rest = torch.ones(kc.shape[0] * page, dtype=torch.bool, device="cuda")
    rest[to] = False
    assert torch.equal(kc.view(-1, hk, d)[rest], x["kc"].view(-1, hk, d)[rest])
    assert torch.equal(vc.view(-1, hk, d)[rest], x["vc"].view(-1, hk, d)[rest])


def test_bad_slots_and_positions_inside_a_walk(cuda_device):
    """Reported, and the tokens around them are as they would be."""
    t, hq, hk, d, page = 8190, 16, 2, 256, 64
    x = make(9, t, hq, hk, d, page, -(-t // page), 64)
    first = x["kc"].clone()
    x["slots"][5::97] = x["kc"].shape[0] * page + 3
    x["positions"][2::89] = 1000
    x["positions"][3::89] = -1
    gdnr.read_device_error()
    q = gdnr.qk_norm_rope_append(x["q"], x["k"], x["v"], x["positions"], x["slots"], x["table"], x["kc"], x["vc"])
    assert gdnr.read_device_error() == 0x8 | 0x2
    inside = (x["positions"] >= 0) & (x["positions"] < 1000)
    rows = x["table"][x["positions"].clamp(0, 999).long()]
    wq, wk = (torch.where(inside[:, None, None], R.norm_rope(y, None, 0, 0, rows, False), y.double()) for y in (x["q"], x["k"]))
    near(q, wq)
    kept = x["slots"] < x["kc"].shape[0] * page
    near(x["kc"].view(-1, hk, d)[x["slots"][kept].long()], wk[kept])
    rest = torch.ones(x["kc"].shape[0] * page, dtype=torch.bool, device="cuda")
    rest[x["slots"][kept].long()] = False
    assert torch.equal(x["kc"].view(-1, hk, d)[rest], first.view(-1, hk, d)[rest])


def test_in_place_and_strided_caches(cuda_device):
    """q_out is q, a view of the packed projection; K and V interleaved in one buffer, the head before the row."""
    t, hq, hk, d, page, pages = 8001, 8, 2, 128, 32, 260
    x = make(10, t, hq, hk, d, page, pages, 128)
    want = R.norm_rope(x["q"], x["qw"], 0, 1e-6, x["table"][x["positions"].long()], False)
    k = R.norm_rope(x["k"], x["kw"], 0, 1e-6, x["table"][x["positions"].long()], False)
    v = x["v"].clone()
    buf = torch.zeros(pages, 2, hk, page, d, dtype=torch.bfloat16, device="cuda")
    kc, vc = buf[:, 0].transpose(1, 2), buf[:, 1].transpose(1, 2)
    gdnr.qk_norm_rope_append(x["q"], x["k"], x["v"], x["positions"], x["slots"], x["table"], kc, vc, q_weight=x["qw"], k_weight=x["kw"], q_out=x["q"])
    s = x["slots"].long()
    near(x["q"], want)
    near(kc[s // page, s % page], k)
    assert torch.equal(vc[s // page, s % page], v) and torch.equal(x["v"], v)
