"""gdn_prefill against the recurrence in float64.

Tolerances (relative 2-norm).  State: float32 throughout, the bound of every
float32 result here (1e-5).  out: bf16 rounding is 1.7e-3 rms; the stored value and up
to three bf16 operands behind it (state, weights, new values) add in quadrature to
3.4e-3, so 5e-3.
"""

import numpy as np
import pytest
import torch

import gdnr
import hybrid_ref as R

pytestmark = pytest.mark.gpu

TOL_STATE, TOL_OUT = 1e-5, 5e-3


def inputs(seed, lens, h, hv, ab=torch.bfloat16, slots=None, decay="strong"):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = sum(lens)

    def n(*s):
        return torch.randn(*s, generator=g, device="cuda")

    a_log = torch.log(1 + 15 * torch.rand(hv, generator=g, device="cuda")) if decay == "strong" else torch.full((hv,), -4.0, device="cuda")
    return dict(mixed=n(t, 2 * h * 128 + hv * 128).to(torch.bfloat16), a=n(t, hv).to(ab), b=n(t, hv).to(ab), a_log=a_log,
                dt_bias=0.5 * n(hv), state=0.05 * n(slots or len(lens), hv, 128, 128))


def check(d, lens, fresh=None, indices=None, max_seqlen=None, out=None, state=None):
    fresh = [False] * len(lens) if fresh is None else fresh
    rows = list(range(len(lens))) if indices is None else indices
    state = d["state"].clone() if state is None else state
    before = state.clone()
    gdnr.read_device_error()
    got = gdnr.gdn_prefill(
        d["mixed"], d["a"], d["b"], d["a_log"], d["dt_bias"], state, R.cu(lens),
        state_indices=None if indices is None else torch.tensor(indices, dtype=torch.int32, device="cuda"),
        has_initial_state=torch.tensor([not f for f in fresh], device="cuda"),
        max_seqlen=max(lens, default=0) if max_seqlen is None else max_seqlen, out=out)
    assert gdnr.read_device_error() == 0
    live = [i for i, r in enumerate(rows) if indices is None or r > 0]
    want, final = R.gdn(d["mixed"], d["a"], d["b"], d["a_log"], d["dt_bias"], before[[max(rows[i], 0) for i in range(len(lens))]], lens, fresh)
    start = np.cumsum([0] + list(lens))
    for i in range(len(lens)):
        o = got[start[i]:start[i + 1]]
        if i in live:
            if lens[i]:
                assert R.rel(o, want[start[i]:start[i + 1]]) < TOL_OUT, (i, lens[i])
            if lens[i] or fresh[i]:
                assert torch.isfinite(state[rows[i]]).all()
                assert float((state[rows[i]].double() - final[i]).norm()) <= TOL_STATE * float(final[i].norm()), (i, lens[i])
            else:
                assert torch.equal(state[rows[i]], before[rows[i]])
        else:
            assert (o == 0).all()
    untouched = sorted(set(range(len(state))) - {rows[i] for i in live})
    assert torch.equal(state[untouched], before[untouched])
    return got, state


@pytest.mark.parametrize("h,hv", [(16, 32), (2, 2), (1, 4), (3, 3), (2, 6)])
@pytest.mark.parametrize("lens", [[1], [1, 1, 1], [2, 7, 1, 5], [16, 17, 63], [64, 65, 127, 128, 129], [200, 0, 3]])
def test_lengths_and_head_layouts(cuda_device, lens, h, hv):
    d = inputs(len(lens) * 100 + hv, lens, h, hv)
    check(d, lens, fresh=[i % 2 == 1 for i in range(len(lens))])


@pytest.mark.parametrize("hint", [0, 1, 4096])
def test_result_does_not_depend_on_the_length_hint(cuda_device, hint):
    lens = [5, 90, 1]
    check(inputs(3, lens, 2, 4), lens, max_seqlen=hint)


@pytest.mark.parametrize("decay", ["strong", "weak"])
def test_long_sequence(cuda_device, decay):
    lens = [1003]
    check(inputs(4, lens, 2, 4, decay=decay), lens, fresh=[True])


def test_weak_decay_correlated_keys(cuda_device):
    """Keys that repeat and beta near one: the chunk's triangular system is far from the identity."""
    lens = [150, 64]
    d = inputs(5, lens, 2, 4, decay="weak")
    d["mixed"][:, 256:512] = d["mixed"][:1, 256:512] + 0.2 * d["mixed"][:, 256:512]
    d["b"].fill_(4.0)
    check(d, lens, fresh=[True, False])


@pytest.mark.parametrize("ab", [torch.float32, torch.float16])
def test_gate_types(cuda_device, ab):
    lens = [70, 3]
    check(inputs(6, lens, 2, 4, ab=ab), lens)


@pytest.mark.parametrize("lens", [[3, 1, 4, 2], [80, 3, 100, 64]])
def test_state_slots_null_and_out_of_range(cuda_device, lens):
    d = inputs(7, lens, 2, 4, slots=6)
    check(d, lens, indices=[4, 0, 1, 3], fresh=[False, False, True, False])
    state = d["state"].clone()
    got = gdnr.gdn_prefill(d["mixed"], d["a"], d["b"], d["a_log"], d["dt_bias"], state, R.cu(lens), max_seqlen=max(lens),
                           state_indices=torch.tensor([2, 6, -1, 0], dtype=torch.int32, device="cuda"))
    assert gdnr.read_device_error() & 0x8  # GDNR_DEVERR_BAD_SLOT
    assert (got[lens[0]:] == 0).all() and torch.equal(state[3:], d["state"][3:]) and torch.equal(state[:2], d["state"][:2])


@pytest.mark.parametrize("lens", [[2, 1], [75, 64]])
def test_strided_inputs_and_outputs(cuda_device, lens):
    d = inputs(8, lens, 2, 4)
    t = sum(lens)
    wide = torch.zeros(t, d["mixed"].shape[1] + 64, dtype=torch.bfloat16, device="cuda")
    wide[:, 32:-32] = d["mixed"]
    d["mixed"] = wide[:, 32:-32]
    ab = torch.stack([d["a"], d["b"]], -1)
    d["a"], d["b"] = ab[..., 0], ab[..., 1]
    d["a_log"] = torch.stack([d["a_log"]] * 3, 1)[:, 1]
    big = torch.full((t, 5, 136), float("nan"), dtype=torch.bfloat16, device="cuda")
    pool = torch.full((len(lens), 6, 128, 128), 7.0, device="cuda")
    pool[:, 1:5] = d["state"]
    check(d, lens, out=big[:, 1:, :128], state=pool[:, 1:5])
    assert torch.isnan(big[:, 0]).all() and torch.isnan(big[..., 128:]).all()
    assert (pool[:, 0] == 7).all() and (pool[:, 5] == 7).all()


def test_parts_of_a_prompt_equal_the_whole(cuda_device):
    """200 tokens at once, and as 100 + 37 + 1 + 62 on the carried state."""
    d = inputs(9, [200], 2, 4)
    _, whole = check(d, [200], fresh=[True])
    state = torch.full_like(d["state"], float("nan"))
    at = 0
    for i, m in enumerate([100, 37, 1, 62]):
        s = slice(at, at + m)
        gdnr.gdn_prefill(d["mixed"][s], d["a"][s], d["b"][s], d["a_log"], d["dt_bias"], state, R.cu([m]), max_seqlen=m,
                         has_initial_state=torch.tensor([i > 0], device="cuda"))
        at += m
    assert R.rel(state, whole) < 2 * TOL_STATE  # two results, each within TOL_STATE of the recurrence


def test_extreme_gates(cuda_device):
    """Decay to nothing in one token, no decay at all, beta of zero and one."""
    lens = [130, 2]
    d = inputs(10, lens, 2, 4)
    d["a_log"] = torch.tensor([2.7, -30.0, 2.7, -30.0], device="cuda")
    d["a"][::3] = 30.0
    d["a"][1::3] = -60.0
    d["b"][::2] = 40.0
    d["b"][1::4] = -40.0
    check(d, lens)


def test_zero_keys_and_queries(cuda_device):
    lens = [66, 2]
    d = inputs(11, lens, 2, 4)
    d["mixed"][::5, :512] = 0
    check(d, lens)


def test_slot_offsets_past_32_bits(cuda_device):
    lens = [2, 70]
    slots = 2 ** 31 // (32 * 128 * 128) + 2
    d = inputs(12, lens, 16, 32, slots=2)
    pool = torch.empty(slots, 32, 128, 128, device="cuda")
    rows = [slots - 1, slots - 2]
    for i, r in enumerate(rows):
        pool[r] = d["state"][i]
    gdnr.gdn_prefill(d["mixed"], d["a"], d["b"], d["a_log"], d["dt_bias"], pool, R.cu(lens), max_seqlen=70,
                     state_indices=torch.tensor(rows, dtype=torch.int32, device="cuda"))
    _, final = R.gdn(d["mixed"], d["a"], d["b"], d["a_log"], d["dt_bias"], d["state"], lens, [False, False])
    for i, r in enumerate(rows):
        assert R.rel(pool[r], final[i]) < TOL_STATE


def test_side_stream_and_graph(cuda_device):
    lens = [70, 3]
    d = inputs(13, lens, 2, 4)
    _, want = check(d, lens)
    s = torch.cuda.Stream()
    state, cu = d["state"].clone(), R.cu(lens)
    out = torch.empty(sum(lens), 4, 128, dtype=torch.bfloat16, device="cuda")
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            gdnr.gdn_prefill(d["mixed"], d["a"], d["b"], d["a_log"], d["dt_bias"], state, cu, max_seqlen=70, out=out)
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(state, want)


def test_decode_continues_from_a_prefilled_state(cuda_device):
    """Prompt by gdn_prefill, the state to a full-precision ReplayState, one decode step: the next row of the recurrence."""
    m, h, hv = 70, 2, 4
    d = inputs(14, [m + 1], h, hv)
    state = d["state"].clone()
    gdnr.gdn_prefill(d["mixed"][:m], d["a"][:m], d["b"][:m], d["a_log"], d["dt_bias"], state, R.cu([m]), max_seqlen=m)
    st = gdnr.ReplayState.allocate(1, h, hv, 4, checkpoint_dtype=torch.float32)
    st.load_state(state)
    got = st.step(d["mixed"][m:], d["a"][m:], d["b"][m:], d["a_log"], d["dt_bias"])
    want, _ = R.gdn(d["mixed"], d["a"], d["b"], d["a_log"], d["dt_bias"], d["state"], [m + 1], [False])
    assert R.rel(got, want[m:]) < TOL_OUT  # the step's ring rounds q, k to bf16


@pytest.mark.parametrize("lens", [[70], [3]])
def test_gates_of_minus_infinity(cuda_device, lens):
    """A decay so strong that its logarithm overflows float32 clears the state; nothing turns into NaN."""
    d = inputs(15, lens, 2, 4)
    d["a_log"] = torch.full((4,), 80.0, device="cuda")  # exp(80) softplus(20) = 1e36, times 3e38 / 20 below: infinite
    d["a"][::2] = 3.0e38
    d["a"][1::2] = -200.0  # softplus underflows: no decay
    check(d, lens)


def test_many_sequences(cuda_device):
    lens = [1 + (7 * i) % 90 for i in range(60)]
    check(inputs(16, lens, 1, 2), lens, fresh=[i % 3 == 0 for i in range(60)])


@pytest.mark.parametrize("lens,h,hv", [([70, 200], 2, 4), ([3, 1], 2, 4), ([64, 70, 130, 64, 90, 64, 65, 64, 100, 64], 16, 32)])
@pytest.mark.parametrize("b", [-200.0, -85.0])
def test_nothing_written_beside_a_large_state(cuda_device, lens, h, hv, b):
    """beta of zero, or next to it, and outputs of hundreds: what is written and what is read differ by 2^100 and more."""
    d = inputs(17, lens, h, hv, decay="weak")
    d["b"].fill_(b)
    d["state"] *= 20000
    check(d, lens)


@pytest.mark.parametrize("lens,h,hv", [([70, 130], 2, 4), ([3, 1], 2, 4), ([64, 70, 130, 64, 90, 64, 65, 64, 100, 64], 16, 32)])
@pytest.mark.parametrize("part", ["all", "values and some queries", "keys"])
def test_zeros(cuda_device, lens, h, hv, part):
    """What a dry run gives: nothing is written and nothing read, but norms of zero have factors of up to 1e3."""
    d = inputs(18, lens, h, hv)
    if part == "all":
        d["mixed"].zero_()
    elif part == "keys":
        d["mixed"][:, h * 128:2 * h * 128] = 0
    else:
        d["mixed"][:, 2 * h * 128:] = 0
        d["mixed"][::3, :h * 128] = 0
    d["state"].zero_()
    got, state = check(d, lens)
    assert (got == 0).all() and (state == 0).all()


@pytest.mark.parametrize("lens,h,hv", [([70, 130], 2, 4), ([3, 1], 2, 4), ([64, 70, 130, 64, 90, 64, 65, 64, 100, 64], 16, 32)])
def test_small_state_and_no_values(cuda_device, lens, h, hv):
    """A state far below one, still far inside float32's range, that the tokens only correct: as exact as any other."""
    d = inputs(19, lens, h, hv, decay="weak")
    d["mixed"][:, 2 * h * 128:] = 0
    d["state"] *= 1e-25
    check(d, lens)


@pytest.mark.parametrize("lens,h,hv", [([64, 128, 70], 2, 4), ([19, 7], 2, 4), ([64, 70, 130, 64, 90, 64, 65, 64, 100, 64], 16, 32)])
def test_little_written_behind_large_values(cuda_device, lens, h, hv):
    """The last tokens of each sequence write 1e-4 of what the ones before them did, which has decayed: the state is theirs.
    Entries of the chunk's system count to 2^-39 there and values to 2^-34 of the largest, 1e-6 of such a state."""
    d = inputs(20, lens, h, hv)
    end = 0
    for m in lens:
        end += m
        d["mixed"][end - min(m // 2, 40):end, 2 * h * 128:] *= 1e-4
    check(d, lens)
