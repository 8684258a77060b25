"""paged_attention on lengths and values that are not in order, in each of its forms.  Inputs and tolerances are
test_gpu_paged_attention.py's.
"""

import pytest
import torch

import gdnr
import hybrid_ref as R
from test_gpu_paged_attention import TOL_LSE, TOL_OUT, check, make

pytestmark = pytest.mark.gpu

# tokens of each sequence, their lengths, page size: few rows by TMA, pages of any size (few and many rows), few rows cut between
# shares, many rows, both kinds
FORMS = [([1, 1], [70, 300], 16), ([3, 2], [70, 301], 5), ([90, 2], [170, 301], 5), ([1, 2], [5000, 9000], 64), ([150, 70], [190, 333], 16),
         ([1, 200], [2000, 260], 32)]


@pytest.mark.parametrize("q_lens,kv_lens,page", FORMS)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_nan_in_a_row_or_a_key(cuda_device, q_lens, kv_lens, page, d):
    """Whoever sees it has NaN in out and lse, nobody else: the rows before a key's place do not."""
    x = make(13, q_lens, kv_lens, 8, 2, d, page)
    want, low = R.attention(x["q"], x["kc"], x["vc"], x["table"], x["kv"], q_lens, d ** -0.5)
    bad = torch.zeros(want.shape[:2], dtype=torch.bool, device="cuda")
    x["q"][0, 3, 7] = float("nan")
    bad[0, 3] = True
    place = kv_lens[1] - 1
    x["kc"][x["table"][1, place // page].long(), place % page, 1, 5] = float("nan")
    bad[sum(q_lens) - 1, 4:] = True
    out, lse = gdnr.paged_attention(x["q"], x["kc"], x["vc"], x["table"], x["kv"], R.cu(q_lens), max_seqlen=max(q_lens), return_lse=True)
    assert torch.equal(torch.isnan(lse), bad)
    assert torch.equal(torch.isnan(out).all(-1), bad) and torch.equal(torch.isnan(out).any(-1), bad)
    assert R.rel(out[~bad], want[~bad]) < TOL_OUT and float((lse.double() - low)[~bad].abs().max()) < TOL_LSE


@pytest.mark.parametrize("q_lens,kv_lens,page", FORMS)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_length_outside_the_block_table_is_reported(cuda_device, q_lens, kv_lens, page, d):
    """One past the table, far past it, below zero: reported, and computed with the nearest length that is in order."""
    for wrong in (1, 2 ** 31 - 1, -1):
        x = make(12, q_lens, kv_lens, 8, 2, d, page)
        full = x["table"].shape[1] * page
        x["table"].clamp_(min=0)
        x["kv"][1] = full if wrong > 0 else 0
        want, low = check(x)
        x["kv"][1] = min(full + wrong, 2 ** 31 - 1) if wrong > 0 else wrong
        gdnr.read_device_error()
        out, lse = gdnr.paged_attention(x["q"], x["kc"], x["vc"], x["table"], x["kv"], R.cu(q_lens), max_seqlen=max(q_lens), return_lse=True)
        assert gdnr.read_device_error() == 0x8
        assert torch.equal(out, want) and torch.equal(lse, low)
