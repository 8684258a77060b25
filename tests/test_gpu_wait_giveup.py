"""A bounded wait that gives up while the other warps' waits are met: all consumers leave together, the copies in flight
land before their warp leaves, and the context stays usable.  tests/wait_giveup.cu has the kernel, built here.
"""

import ctypes
import pathlib
import shutil
import subprocess
import time

import pytest
import torch

from gdnr import _lib

pytestmark = pytest.mark.gpu

HERE = pathlib.Path(__file__).resolve().parent
CSRC = HERE.parent / "fp8-replayssm-gdn-kernel_b200" / "csrc"


@pytest.mark.skipif(shutil.which("nvcc") is None, reason="nvcc not available")
def test_consumers_leave_together_and_copies_land(cuda_device, tmp_path):
    lib = tmp_path / "wait_giveup.so"
    subprocess.run(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O2", "-shared", "-Xcompiler", "-fPIC", "-I", str(CSRC),
                    str(HERE / "wait_giveup.cu"), "-o", str(lib)], check=True)
    run = ctypes.CDLL(str(lib)).run
    run.argtypes = [ctypes.c_void_p] * 3
    src = torch.arange(8192, dtype=torch.int32, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    report = torch.full((9,), -1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    t = time.perf_counter()
    assert run(src.data_ptr(), err.data_ptr(), report.data_ptr()) == 0
    torch.cuda.synchronize()
    assert 0.9 < time.perf_counter() - t < 5  # one limit of 1 s
    assert int(err.item()) == _lib.DEVERR_WAIT_TIMEOUT
    report = report.tolist()
    assert report[:4] == [0, 1, 1, 1]  # only the first warp's wait gave up
    assert report[4:8] == [1, 1, 1, 1]  # all left, none met the barrier behind
    assert report[8] == 0  # both tiles had landed when the requesting warp left
