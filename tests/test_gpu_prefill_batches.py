"""gdn_prefill on batches with many heads in all, whose sequences take a multiprocessor a head
(test_gpu_prefill.py has few heads: four multiprocessors a head).  Inputs, checks and tolerances are that file's.
"""

import pytest
import torch

import gdnr
import hybrid_ref as R
from test_gpu_prefill import TOL_STATE, check, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("h,hv", [(16, 32), (32, 32), (8, 32), (10, 30), (4, 24)])
def test_ragged_batch(cuda_device, h, hv):
    lens = [64, 65, 127, 1, 200, 0, 3, 128, 63, 31, 257, 17]
    check(inputs(100 + h, lens, h, hv), lens, fresh=[i % 3 == 1 for i in range(len(lens))])


@pytest.mark.parametrize("decay", ["strong", "weak"])
def test_one_long_sequence_among_short_ones(cuda_device, decay):
    lens = [100] * 5 + [1003] + [100] * 6
    check(inputs(110, lens, 16, 32, decay=decay), lens, fresh=[i == 5 for i in range(len(lens))])


def test_weak_decay_correlated_keys(cuda_device):
    lens = [150, 64, 70, 31, 64, 64, 130, 64, 90, 64]
    d = inputs(111, lens, 16, 32, decay="weak")
    keys = slice(16 * 128, 32 * 128)
    d["mixed"][:, keys] = d["mixed"][:1, keys] + 0.2 * d["mixed"][:, keys]
    d["b"].fill_(4.0)
    check(d, lens, fresh=[i % 2 == 0 for i in range(len(lens))])


@pytest.mark.parametrize("ab", [torch.float32, torch.float16])
def test_gate_types(cuda_device, ab):
    lens = [70] * 10
    check(inputs(112, lens, 16, 32, ab=ab), lens)


def test_state_slots_null_and_out_of_range(cuda_device):
    lens = [80, 3, 100, 64, 77, 0, 65, 64, 129, 90]
    indices = [12, 0, 1, 3, 9, 2, 0, 7, 5, 10]
    d = inputs(113, lens, 16, 32, slots=13)
    check(d, lens, indices=indices, fresh=[i in (2, 5) for i in range(10)])
    indices[3], indices[8] = 13, -1
    state = d["state"].clone()
    got = gdnr.gdn_prefill(d["mixed"], d["a"], d["b"], d["a_log"], d["dt_bias"], state, R.cu(lens), max_seqlen=max(lens),
                           state_indices=torch.tensor(indices, dtype=torch.int32, device="cuda"))
    assert gdnr.read_device_error() & 0x8  # GDNR_DEVERR_BAD_SLOT
    assert (got[183:247] == 0).all() and (got[453:582] == 0).all()
    kept = [0, 2, 3, 4, 5, 6, 8, 11]
    assert torch.equal(state[kept], d["state"][kept])


def test_strided_inputs_and_outputs(cuda_device):
    lens = [75, 64, 80, 64, 100, 70, 64, 65]
    d = inputs(114, lens, 16, 32)
    t = sum(lens)
    wide = torch.zeros(t, d["mixed"].shape[1] + 64, dtype=torch.bfloat16, device="cuda")
    wide[:, 32:-32] = d["mixed"]
    d["mixed"] = wide[:, 32:-32]
    ab = torch.stack([d["a"], d["b"]], -1)
    d["a"], d["b"] = ab[..., 0], ab[..., 1]
    big = torch.full((t, 33, 136), float("nan"), dtype=torch.bfloat16, device="cuda")
    pool = torch.full((len(lens), 34, 128, 128), 7.0, device="cuda")
    pool[:, 1:33] = d["state"]
    check(d, lens, out=big[:, 1:, :128], state=pool[:, 1:33])
    assert torch.isnan(big[:, 0]).all() and torch.isnan(big[..., 128:]).all()
    assert (pool[:, 0] == 7).all() and (pool[:, 33] == 7).all()


def test_other_sequences_garbage_stays_theirs(cuda_device):
    """A chunk's tile reads past its sequence's end: NaN there must not come in."""
    lens = [70, 64, 33, 100, 64, 65, 90, 64, 64, 64]
    d = inputs(115, lens, 16, 32)
    clean, _ = check(d, lens)
    d["mixed"][70:134] = float("nan")
    got = gdnr.gdn_prefill(d["mixed"], d["a"], d["b"], d["a_log"], d["dt_bias"], d["state"].clone(), R.cu(lens), max_seqlen=max(lens))
    assert torch.equal(got[:70], clean[:70]) and torch.equal(got[134:], clean[134:])


def test_gates_of_minus_infinity(cuda_device):
    lens = [70, 64, 128, 65, 64, 64, 80, 64, 64, 64]
    d = inputs(116, lens, 16, 32)
    d["b"][20:40] = float("-inf")
    d["a"][75:80] = float("-inf")
    check(d, lens)


def test_parts_of_a_prompt_equal_the_whole(cuda_device):
    """Ten prompts of 200 tokens at once, and as 128 + 72 on the carried states."""
    n = 10
    d = inputs(117, [200] * n, 16, 32)
    _, whole = check(d, [200] * n, fresh=[True] * n)
    state = torch.full_like(d["state"], float("nan"))
    rows = torch.arange(200 * n, device="cuda").reshape(n, 200)
    for i, s in enumerate([slice(0, 128), slice(128, 200)]):
        r = rows[:, s].reshape(-1)
        m = r.numel() // n
        gdnr.gdn_prefill(d["mixed"][r], d["a"][r], d["b"][r], d["a_log"], d["dt_bias"], state, R.cu([m] * n), max_seqlen=m,
                         has_initial_state=torch.tensor([i > 0] * n, device="cuda"))
    assert R.rel(state, whole) < 2 * TOL_STATE  # two results, each within TOL_STATE of the recurrence


def test_same_result_every_time(cuda_device):
    lens = [200, 64, 130, 64, 70, 64, 64, 65, 64, 64]
    d = inputs(118, lens, 16, 32)
    first, state = check(d, lens)
    for _ in range(3):
        again, other = check(d, lens)
        assert torch.equal(first, again) and torch.equal(state, other)


def test_stages_are_used_again_many_times(cuda_device):
    """Twenty chunks a sequence through three stages, each chunk's output laid over its values before the next ones arrive there;
    values of very different sizes from chunk to chunk, so that one that is not its own shows."""
    lens = [1280, 1217, 1150, 1030, 1279, 1111, 1283, 1024]
    d = inputs(119, lens, 16, 32)
    t = torch.arange(sum(lens), device="cuda") // 64
    d["mixed"][:, 32 * 128:] *= torch.tensor([1.0, 64.0, 0.25, 8.0, 512.0], device="cuda")[t % 5][:, None].bfloat16()
    first, state = check(d, lens)
    for _ in range(10):
        again = d["state"].clone()
        got = gdnr.gdn_prefill(d["mixed"], d["a"], d["b"], d["a_log"], d["dt_bias"], again, R.cu(lens), max_seqlen=max(lens))
        assert torch.equal(first, got) and torch.equal(state, again)


@pytest.mark.parametrize("h,hv,lens", [(16, 32, [70, 64, 128, 65, 64, 64, 80, 64, 64, 64]), (2, 4, [70, 64, 150])])
def test_decay_that_clears_the_state(cuda_device, h, hv, lens):
    """Gates of minus infinity, several in a row and at the borders of chunks and of their 16-token blocks: what came before such
    a token is gone, nothing turns into NaN, also for the whole inverse of the chunk's system."""
    d = inputs(120, lens, h, hv)
    d["a_log"] = torch.full((hv,), 80.0, device="cuda")  # exp(80) softplus(3e38) is infinite
    d["a"].fill_(-200.0)  # softplus underflows: no decay
    for t in (0, 15, 16, 17, 31, 48, 63, 64, 69, 70, 100, 133, 134, 140, 200, sum(lens) - 1):
        d["a"][t] = 3.0e38
    got, state = check(d, lens)
    cleared = d["state"].clone() * 1e6
    again = gdnr.gdn_prefill(d["mixed"], d["a"], d["b"], d["a_log"], d["dt_bias"], cleared, R.cu(lens), max_seqlen=max(lens))
    assert torch.equal(again[:70], got[:70]) and torch.equal(cleared[0], state[0])  # its first token clears the state


def test_other_sequences_garbage_stays_theirs_with_few_heads(cuda_device):
    """As above on the scan that spreads a head over multiprocessors."""
    lens = [70, 64, 33, 100]
    d = inputs(121, lens, 2, 4)
    clean, _ = check(d, lens)
    d["mixed"][70:134] = float("nan")
    got = gdnr.gdn_prefill(d["mixed"], d["a"], d["b"], d["a_log"], d["dt_bias"], d["state"].clone(), R.cu(lens), max_seqlen=max(lens))
    assert torch.equal(got[:70], clean[:70]) and torch.equal(got[134:], clean[134:])
