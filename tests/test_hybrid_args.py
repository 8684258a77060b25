"""The prompt operators' refusals and argument structures, without a GPU: nothing here launches."""

import ctypes
import pathlib
import shutil
import subprocess

import pytest
import torch

import gdnr
from gdnr import _lib

FAKE = 0x10000  # 16-byte aligned, never dereferenced


def desc(shape, dtype, stride=None, data=FAKE):
    d = _lib.Tensor()
    d.data, d.dtype, d.ndim = data, dtype, len(shape)
    if stride is None:
        stride, acc = [], 1
        for s in reversed(shape):
            stride.insert(0, acc)
            acc *= s
    for i, (s, st) in enumerate(zip(shape, stride)):
        d.shape[i], d.stride[i] = s, st
    return d


def refuse(name, args, code, needle):
    lib = _lib.load()
    rc = getattr(lib, name)(bytes(args), None)
    msg = lib.gdnr_last_error().decode()
    assert rc == code and needle in msg, (rc, msg)


def prefill(t=5, n=2, h=2, hv=4, **over):
    a = _lib.PrefillArgs()
    far = 1 << 40
    a.mixed_qkv = desc([t, 256 * h + 128 * hv], _lib.BF16)
    a.a, a.b = desc([t, hv], _lib.BF16), desc([t, hv], _lib.BF16)
    a.a_log, a.dt_bias = desc([hv], _lib.F32), desc([hv], _lib.F32)
    a.state = desc([n, hv, 128, 128], _lib.F32, data=far)
    a.cu_seqlens = desc([n + 1], _lib.I32)
    a.out = desc([t, hv, 128], _lib.BF16, data=2 * far)
    a.error_flag = FAKE
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,code,needle", [
    (dict(state=desc([2, 4, 64, 64], _lib.F32)), _lib.ERR_UNSUPPORTED, "V = 128"),
    (dict(state=desc([2, 4, 128, 128], _lib.BF16)), _lib.ERR_DTYPE, "state"),
    (dict(state=desc([1, 4, 128, 128], _lib.F32, data=1 << 40)), _lib.ERR_ARG, "slots"),
    (dict(state=desc([2, 4, 128, 128], _lib.F32, stride=[70000, 17000, 132, 1])), _lib.ERR_LAYOUT, "packed"),
    (dict(state=desc([2, 4, 128, 128], _lib.F32, data=FAKE + 4)), _lib.ERR_LAYOUT, "16-byte"),
    (dict(mixed_qkv=desc([5, 1000], _lib.BF16)), _lib.ERR_ARG, "mixed_qkv"),
    (dict(mixed_qkv=desc([5, 1024], _lib.F32)), _lib.ERR_DTYPE, "mixed_qkv"),
    (dict(mixed_qkv=desc([5, 1024], _lib.BF16, stride=[1028, 1])), _lib.ERR_LAYOUT, "mixed_qkv"),
    (dict(mixed_qkv=desc([5, 3 * 256 + 512], _lib.BF16)), _lib.ERR_ARG, "multiple of H"),
    (dict(a=desc([5, 3], _lib.BF16)), _lib.ERR_ARG, "a:"),
    (dict(cu_seqlens=desc([0], _lib.I32)), _lib.ERR_ARG, "cu_seqlens"),
    (dict(cu_seqlens=desc([3], _lib.F32)), _lib.ERR_DTYPE, "cu_seqlens"),
    (dict(state_indices=desc([3], _lib.I32)), _lib.ERR_ARG, "state_indices"),
    (dict(has_initial=desc([2], _lib.I32)), _lib.ERR_DTYPE, "has_initial"),
    (dict(out=desc([5, 4, 128], _lib.F32)), _lib.ERR_DTYPE, "out"),
    (dict(out=desc([5, 4, 128], _lib.BF16)), _lib.ERR_ALIAS, "out"),
    (dict(max_seqlen=-1), _lib.ERR_ARG, "max_seqlen"),
])
def test_prefill_refusals(over, code, needle):
    refuse("gdnr_gdn_prefill", prefill(**over), code, needle)


def append(t=5, hq=4, hk=2, d=128, **over):
    a = _lib.AppendArgs()
    far = 1 << 40
    a.q, a.k, a.v = desc([t, hq, d], _lib.BF16), desc([t, hk, d], _lib.BF16), desc([t, hk, d], _lib.BF16)
    a.positions, a.slots = desc([t], _lib.I32), desc([t], _lib.I32)
    a.cos_sin = desc([100, min(d, 64)], _lib.F32)
    a.q_out = desc([t, hq, d], _lib.BF16, data=far)
    a.k_cache, a.v_cache = desc([3, 16, hk, d], _lib.BF16, data=2 * far), desc([3, 16, hk, d], _lib.BF16, data=3 * far)
    a.eps = 1e-6
    a.error_flag = FAKE
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,code,needle", [
    (dict(d=96), _lib.ERR_UNSUPPORTED, "head dim"),
    (dict(q=desc([5, 4, 128], _lib.F32)), _lib.ERR_DTYPE, "q:"),
    (dict(q=desc([5, 4, 128], _lib.BF16, stride=[512, 128, 2])), _lib.ERR_LAYOUT, "innermost"),
    (dict(k=desc([5, 2, 64], _lib.BF16)), _lib.ERR_ARG, "k:"),
    (dict(v=desc([5, 1, 128], _lib.BF16)), _lib.ERR_ARG, "v:"),
    (dict(q_weight=desc([64], _lib.BF16)), _lib.ERR_ARG, "q_weight"),
    (dict(k_weight=desc([128], _lib.F16)), _lib.ERR_DTYPE, "k_weight"),
    (dict(cos_sin=desc([100, 130], _lib.F32)), _lib.ERR_ARG, "cos_sin"),
    (dict(cos_sin=desc([100, 7], _lib.F32)), _lib.ERR_ARG, "cos_sin"),
    (dict(slots=desc([4], _lib.I32)), _lib.ERR_ARG, "slots"),
    (dict(k_cache=desc([3, 16, 4, 128], _lib.BF16)), _lib.ERR_ARG, "k_cache"),
    (dict(v_cache=desc([3, 8, 2, 128], _lib.BF16)), _lib.ERR_ARG, "v_cache"),
    (dict(k_cache=desc([3, 0, 2, 128], _lib.BF16), v_cache=desc([3, 0, 2, 128], _lib.BF16)), _lib.ERR_ARG, "page_size"),
    (dict(q_out=desc([5, 4, 128], _lib.BF16, data=FAKE + 32)), _lib.ERR_ALIAS, "q_out"),
    (dict(v_cache=desc([3, 16, 2, 128], _lib.BF16, data=2 << 40)), _lib.ERR_ALIAS, "k_cache"),
    (dict(eps=float("nan")), _lib.ERR_ARG, "eps"),
    (dict(interleaved=2), _lib.ERR_ARG, "interleaved"),
])
def test_append_refusals(over, code, needle):
    refuse("gdnr_qk_norm_rope_append", append(**over), code, needle)


def attn(t=5, n=2, hq=4, hk=2, d=128, **over):
    a = _lib.AttnArgs()
    far = 1 << 40
    a.q = desc([t, hq, d], _lib.BF16)
    a.k_cache, a.v_cache = desc([3, 16, hk, d], _lib.BF16), desc([3, 16, hk, d], _lib.BF16)
    a.block_table, a.kv_lens, a.cu_seqlens = desc([n, 2], _lib.I32), desc([n], _lib.I32), desc([n + 1], _lib.I32)
    a.out = desc([t, hq, d], _lib.BF16, data=far)
    a.scale = 0.1
    a.error_flag = FAKE
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over,code,needle", [
    (dict(d=80), _lib.ERR_UNSUPPORTED, "head dim"),
    (dict(hq=5), _lib.ERR_ARG, "multiple of Hk"),
    (dict(q=desc([5, 4, 128], _lib.F16)), _lib.ERR_DTYPE, "q:"),
    (dict(k_cache=desc([3, 16, 2, 64], _lib.BF16)), _lib.ERR_ARG, "k_cache"),
    (dict(v_cache=desc([3, 16, 2, 128], _lib.BF16, stride=[4100, 256, 128, 1])), _lib.ERR_LAYOUT, "v_cache"),
    (dict(block_table=desc([3, 2], _lib.I32)), _lib.ERR_ARG, "block_table"),
    (dict(block_table=desc([2, 2], _lib.I32, stride=[4, 2])), _lib.ERR_LAYOUT, "block_table"),
    (dict(kv_lens=desc([1], _lib.I32)), _lib.ERR_ARG, "kv_lens"),
    (dict(cu_seqlens=desc([3], _lib.I32, stride=[2])), _lib.ERR_LAYOUT, "cu_seqlens"),
    (dict(out=desc([5, 4, 128], _lib.BF16)), _lib.ERR_ALIAS, "out"),
    (dict(lse=desc([5, 3], _lib.F32)), _lib.ERR_ARG, "lse"),
    (dict(scale=float("inf")), _lib.ERR_ARG, "scale"),
    (dict(max_seqlen=-2), _lib.ERR_ARG, "max_seqlen"),
    (dict(workspace=None), _lib.ERR_ARG, "workspace"),
    (dict(workspace=FAKE + 8, workspace_bytes=1 << 40), _lib.ERR_ARG, "workspace"),
])
def test_attention_refusals(over, code, needle):
    refuse("gdnr_paged_attention", attn(**over), code, needle)


def test_null_arguments():
    lib = _lib.load()
    for name in ("gdnr_gdn_prefill", "gdnr_qk_norm_rope_append", "gdnr_paged_attention"):
        assert getattr(lib, name)(None, None) == _lib.ERR_ARG


def test_nothing_to_do_is_no_error():
    lib = _lib.load()
    assert lib.gdnr_gdn_prefill(bytes(prefill(t=0, n=0)), None) == _lib.OK
    assert lib.gdnr_qk_norm_rope_append(bytes(append(t=0)), None) == _lib.OK
    assert lib.gdnr_paged_attention(bytes(attn(t=0)), None) == _lib.OK


def test_host_tensors_are_refused():
    z = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        gdnr.paged_attention(z, z[None], z[None], i[None], i, i)
    with pytest.raises(ValueError, match="CUDA"):
        gdnr.qk_norm_rope_append(z, z, z, i, i, torch.zeros(4, 64), z[None], z[None])
    with pytest.raises(ValueError, match="CUDA"):
        gdnr.gdn_prefill(z[:, 0], z[:, 0], z[:, 0], i, i, torch.zeros(1, 1, 128, 128), i)


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_structs_match_c(tmp_path):
    header = pathlib.Path(__file__).resolve().parent.parent / "include"
    structs = {"gdnr_prefill_args": _lib.PrefillArgs, "gdnr_append_args": _lib.AppendArgs, "gdnr_attn_args": _lib.AttnArgs}
    src = tmp_path / "sz.c"
    body = "".join(f'  printf("{n} %zu %zu\\n", sizeof({n}), offsetof({n}, error_flag));\n' for n in structs)
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "gdnr.h"\nint main(void) {{\n{body}  return 0;\n}}\n')
    exe = tmp_path / "sz"
    subprocess.run(["gcc", "-I", str(header), str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        name, size, off = line.split()
        assert int(size) == ctypes.sizeof(structs[name]) and int(off) == structs[name].error_flag.offset


def test_packed_bytes_are_the_structure():
    """The tails that the calls pack against the ctypes structures."""
    from gdnr import hybrid

    for cls, tail, tensors in ((_lib.PrefillArgs, hybrid._PREFILL_TAIL, 10), (_lib.AppendArgs, hybrid._APPEND_TAIL, 11),
                               (_lib.AttnArgs, hybrid._ATTN_TAIL, 8)):
        assert ctypes.sizeof(cls) == tensors * ctypes.sizeof(_lib.Tensor) + tail.size
