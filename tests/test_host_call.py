"""The compiled call path (gdnr/_host.so) on tensors that a kernel must not be given, without a GPU.

Fake tensors say that they are on a CUDA device and have shapes and strides, but no memory."""

import pathlib
import subprocess
import sys

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import gdnr

BF16, I32, F32 = torch.bfloat16, torch.int32, torch.float32


@pytest.fixture
def fake():
    with FakeTensorMode() as mode:
        yield mode


def bf16(*shape):
    return torch.empty(*shape, dtype=BF16, device="cuda:0")


def append_tensors(device="cuda:0"):
    def z(*shape, dtype=BF16):
        return torch.empty(*shape, dtype=dtype, device=device)

    return [z(2, 4, 64), z(2, 2, 64), z(2, 2, 64), z(2, dtype=I32), z(2, dtype=I32), z(9, 64, dtype=F32), z(3, 16, 2, 64), z(3, 16, 2, 64)]


def test_tensor_without_memory_is_refused(fake):
    x = append_tensors()
    with pytest.raises(ValueError, match="argument 0 has elements but no memory"):
        gdnr.qk_norm_rope_append(*x, q_out=x[0])


@pytest.mark.parametrize("name,at", [("q_weight", 3), ("k_weight", 4)])
def test_optional_tensor_without_memory_is_not_taken_for_absent(fake, name, at):
    """The tensors before it are empty ones, which are in order without memory."""
    x = append_tensors()
    empty = [t[:0] for t in x[:5]]
    with pytest.raises(ValueError, match=f"argument {at} has elements but no memory"):
        gdnr.qk_norm_rope_append(*empty, *x[5:], q_out=empty[0], **{name: bf16(64)})


def test_tensors_on_two_devices_are_refused(fake):
    """The first one is empty, so that its missing memory is not what is refused."""
    q, x = bf16(0, 4, 64), append_tensors("cuda:1")
    with pytest.raises(ValueError, match="one device"):
        gdnr.qk_norm_rope_append(q, *x[1:], q_out=q)


IN_A_TRANSFORM = """
import sys
sys.path[:0] = {paths!r}
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
import gdnr
from test_host_call import append_tensors, bf16

with FakeTensorMode():
    x = append_tensors()
    def call(q):
        return gdnr.qk_norm_rope_append(q, *x[1:], q_out=q).sum()
    try:
        {transform}
    except RuntimeError as e:
        print("raised:", str(e).splitlines()[0])
"""


@pytest.mark.parametrize("transform", ["torch.func.grad(call)(x[0])", "torch.func.vmap(call)(bf16(3, 2, 4, 64))"])
def test_a_transform_raises_and_the_process_goes_on(transform):
    """A transform's wrapper has no address: torch throws when it is asked for.  In a process of its own."""
    here = pathlib.Path(__file__).resolve().parent
    paths = [str(here), str(pathlib.Path(gdnr.__file__).resolve().parent.parent)]
    run = subprocess.run([sys.executable, "-c", IN_A_TRANSFORM.format(paths=paths, transform=transform)], capture_output=True, text=True,
                         timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
    assert "raised: Cannot access data pointer" in run.stdout, run.stdout
