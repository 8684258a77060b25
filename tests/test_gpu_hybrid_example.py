"""The example block: prompts at once against the same tokens as shorter prompts and single tokens.

Both ways compute the same function and round at the same places but for the kernels' own
roundings (three bf16 values a layer, 1.7e-3 rms each, and what they move in the second
layer's inputs): 1e-2 relative, with the full-precision checkpoint (no FP8 in between).
"""

import pathlib
import sys

import pytest
import torch

import gdnr
import hybrid_ref as R

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent.parent / "examples"))
import hybrid_prompt as E  # noqa: E402

pytestmark = pytest.mark.gpu


def test_prompt_then_single_tokens_equal_the_whole_prompt(cuda_device):
    sizes, lens, new = E.Sizes(), [37, 1, 130, 64], 9
    block = E.HybridBlock(sizes, seed=1)
    torch.manual_seed(2)
    seqs = [torch.randn(m + new, sizes.width, device="cuda").to(E.BF16) for m in lens]
    whole, _ = E.prefill(block, torch.cat(seqs), [m + new for m in lens], E.PagedCache(sizes, len(lens)))
    ends = torch.tensor([m + new for m in lens]).cumsum(0).tolist()

    gdnr.read_device_error()
    cache = E.PagedCache(sizes, len(lens))
    out, state = E.prefill(block, torch.cat([s[:m] for s, m in zip(seqs, lens)]), lens, cache)
    starts = torch.tensor([0] + lens).cumsum(0).tolist()
    for i, m in enumerate(lens):
        first = ends[i] - m - new
        assert R.rel(out[starts[i]:starts[i + 1]], whole[first:first + m]) < 1e-2
    replay = gdnr.ReplayState.allocate(len(lens), sizes.key_heads, sizes.value_heads, ring_len=4, checkpoint_dtype=torch.float32)
    replay.load_state(state)
    kv_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for t in range(new):
        got = E.decode(block, torch.stack([s[m + t] for s, m in zip(seqs, lens)]), replay, cache, kv_lens)
        want = torch.stack([whole[e - new + t] for e in ends])
        assert R.rel(got, want) < 1e-2, t
    assert gdnr.read_device_error() == 0


def test_example_runs(cuda_device, capsys):
    E.main()
    assert "367 prompt tokens in 4 sequences, 20 tokens each" in capsys.readouterr().out
