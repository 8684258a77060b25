"""paged_attention where the kernel goes by the rows of a sequence (tokens x query heads of a key head): drafts,
mixed batches, short chunks over long contexts.  Inputs, checks and tolerances are test_gpu_paged_attention.py's.
"""

import pytest
import torch

import gdnr
import hybrid_ref as R
from test_gpu_paged_attention import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hk", [(8, 1), (16, 4), (14, 2), (32, 1)])
@pytest.mark.parametrize("page", [8, 24, 64])
@pytest.mark.parametrize("draft", [1, 3, 4, 5, 8])
def test_drafts(cuda_device, d, hq, hk, page, draft):
    """16, 32, 64 rows and the sizes on both sides."""
    kv = [draft, 63, 64, 65, 300, 129, 700]
    check(make(d + hq + page + draft, [draft] * 7, kv, hq, hk, d, page))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hk", [(16, 2), (4, 4), (24, 1), (34, 2)])
@pytest.mark.parametrize("page", [16, 24])
def test_mixed_lengths(cuda_device, d, hq, hk, page):
    q = [1, 1, 65, 2, 1, 200, 3, 0, 1, 17, 33, 1]
    kv = [900, 1, 65, 70, 64, 260, 3, 5, 2000, 400, 33, 0]
    check(make(d + hq + page, q, kv, hq, hk, d, page))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("tokens", [9, 40, 100])
def test_short_chunk_over_a_long_context(cuda_device, d, tokens):
    """One unit cut into dozens of parts."""
    check(make(d + tokens, [tokens], [9001], 16, 2, d, 64))
    check(make(d + tokens, [tokens, tokens - 8], [5001, 4000], 16, 2, d, 64))


@pytest.mark.parametrize("q,kv", [([1] * 40 + [500], [70] * 40 + [900]), ([1, 30, 30], [50, 40, 30]), ([300, 1], [300, 8000])])
def test_one_part_of_a_mixed_batch_is_small(cuda_device, q, kv):
    for d in (128, 256):
        check(make(d, q, kv, 16, 2, d, 16))


def test_mixed_batch_in_a_graph_and_again(cuda_device):
    """Two kernels that overlap and one join: the same result each time, also captured, calls back to back."""
    x = make(7, [1, 90, 1, 300, 2, 1], [500, 90, 2000, 700, 64, 33], 16, 2, 128, 16)
    first, _ = check(x)
    args = x["q"], x["kc"], x["vc"], x["table"], x["kv"], R.cu(x["q_lens"])
    for _ in range(5):
        again = [gdnr.paged_attention(*args, max_seqlen=300) for _ in range(4)]
        assert all(torch.equal(first, y) for y in again)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        out = torch.empty_like(first)
        gdnr.paged_attention(*args, max_seqlen=300, out=out)
        with torch.cuda.graph(graph, stream=stream):
            for _ in range(3):
                gdnr.paged_attention(*args, max_seqlen=300, out=out)
    torch.cuda.synchronize()
    out.fill_(float("nan"))
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
