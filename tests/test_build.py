"""What build.py compiles and links, and when, with the compilers replaced by a recorder."""

import importlib.util
import pathlib
import subprocess
import sys
import types

import pytest
import torch

from gdnr import _lib

CSRC = pathlib.Path(__file__).resolve().parent.parent / "fp8-replayssm-gdn-kernel_b200" / "csrc"


@pytest.fixture
def builder(tmp_path, monkeypatch):
    """build.py with its outputs under tmp_path; ``commands`` are the outputs of what it ran, which are made as empty files."""
    spec = importlib.util.spec_from_file_location("gdnr_build", CSRC / "build.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    commands = []

    def run(cmd, check):
        out = pathlib.Path(cmd[cmd.index("-o") + 1])
        commands.append(out.name)
        out.write_text("")
        return subprocess.CompletedProcess(cmd, 0)

    for name, path in (("BUILD", "_build"), ("TARGET", "libgdnr.so"), ("HOST_TARGET", "_host.so")):
        monkeypatch.setattr(module, name, tmp_path / path)
    monkeypatch.setattr(module, "nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    monkeypatch.setattr(module.subprocess, "run", run)
    module.commands = commands
    return module


def test_everything_once(builder):
    builder.build()
    assert sorted(builder.commands[:-2]) == sorted(p.stem + ".o" for p in CSRC.glob("*.cu"))
    assert builder.commands[-2:] == ["libgdnr.so", "_host.so"]
    builder.commands.clear()
    assert builder.build() == builder.TARGET and builder.commands == []


@pytest.mark.parametrize("without", ["torch", "headers"])
def test_c_library_without_torch(builder, monkeypatch, tmp_path, without):
    if without == "torch":
        monkeypatch.setitem(sys.modules, "torch", None)  # import torch raises
    else:
        monkeypatch.setattr(sys.modules["torch"], "__file__", str(tmp_path / "torch" / "__init__.py"))
    assert builder.build() == builder.TARGET
    assert builder.commands[-1] == "libgdnr.so"


@pytest.mark.parametrize("changed", ["torch", "python"])
def test_host_module_again_after_an_upgrade(builder, monkeypatch, changed):
    builder.build()
    builder.commands.clear()
    if changed == "torch":
        monkeypatch.setattr(torch, "__version__", "99.0")
    else:
        monkeypatch.setattr(builder.sys, "version_info", types.SimpleNamespace(major=9, minor=9))
    builder.build()
    assert builder.commands == ["_host.so"]
    builder.build()
    assert builder.commands == ["_host.so"]


def test_host_module_of_another_torch_is_not_used(monkeypatch):
    """A module that still loads could misread another torch's tensors."""
    assert _lib._host().built_for.startswith(f"torch {torch.__version__},")
    monkeypatch.setattr(_lib, "_host_module", None)
    monkeypatch.setattr(torch, "__version__", "99.0")
    with pytest.raises(RuntimeError, match="build.py.*installed is torch 99.0"):
        _lib._host()
