"""What build.py compiles and links, and when, with the compilers replaced by a recorder."""

import importlib.util
import pathlib
import subprocess
import sys

import pytest
import torch  # noqa: F401

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
