"""Build libgdnr.so (all CUDA sources of this directory) for sm_100a, and the host call path (_host) if there is a torch.

    python fp8-replayssm-gdn-kernel_b200/csrc/build.py [--verbose-ptxas] [--force]

Objects go to ``csrc/_build/``; the shared library is written next to the
Python host package (``gdnr/libgdnr.so``) so that it travels with the tree.
Incremental: a source is recompiled when it or any header is newer than its
object, the host call path also when torch or Python are others than it was built for.
"""

from __future__ import annotations

import argparse
import os
import pathlib
import shutil
import subprocess
import sys
import sysconfig

HERE = pathlib.Path(__file__).resolve().parent
PKG = HERE.parent / "gdnr"
INCLUDE = HERE.parent.parent / "include"
BUILD = HERE / "_build"
TARGET = PKG / "libgdnr.so"
HOST_SOURCE = HERE / "gdnr_host.cpp"
HOST_TARGET = PKG / "_host.so"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-O2", "--expt-relaxed-constexpr"]


def nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found")
    return cand


def build(force: bool = False, verbose_ptxas: bool = False) -> pathlib.Path:
    BUILD.mkdir(exist_ok=True)
    sources = sorted(HERE.glob("*.cu"))
    headers = list(HERE.glob("*.cuh")) + list(HERE.glob("*.h")) + list(INCLUDE.glob("*.h"))
    newest_header = max((h.stat().st_mtime for h in headers), default=0.0)
    objects = []
    for src in sources:
        obj = BUILD / (src.stem + ".o")
        objects.append(obj)
        if (not force and obj.exists() and obj.stat().st_mtime >= src.stat().st_mtime
                and obj.stat().st_mtime >= newest_header):
            continue
        cmd = [nvcc(), *ARCH, *FLAGS, "-I", str(INCLUDE), "-c", str(src), "-o", str(obj)]
        if verbose_ptxas:
            cmd += ["-Xptxas", "-v"]
        print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
    if force or not TARGET.exists() or any(o.stat().st_mtime > TARGET.stat().st_mtime for o in objects):
        cmd = [nvcc(), *ARCH, "-shared", "-o", str(TARGET), *map(str, objects), "-lcuda"]
        print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
    build_host(force)  # last: the C library needs no torch
    return TARGET


def torch_root() -> pathlib.Path | None:
    """The installed torch, if it has its C++ headers."""
    try:
        import torch
    except ImportError:
        return None
    root = pathlib.Path(torch.__file__).resolve().parent
    return root if (root / "include" / "torch").is_dir() else None


def build_host(force: bool = False) -> pathlib.Path | None:
    """gdnr/_host.so: the CPython module over torch's C++ tensors (g++, no device code); None without torch."""
    root = torch_root()
    if root is None:
        print("no torch with C++ headers: gdnr/_host.so (the Python functions of the prompt operators) is not built", flush=True)
        return None
    import torch

    # what the module's import compares (gdnr/_lib.py)
    built_for = f"torch {torch.__version__}, Python {sys.version_info.major}.{sys.version_info.minor}"
    record = BUILD / "host.txt"
    newest = max(HOST_SOURCE.stat().st_mtime, (INCLUDE / "gdnr.h").stat().st_mtime)
    if (not force and HOST_TARGET.exists() and HOST_TARGET.stat().st_mtime >= newest
            and record.exists() and record.read_text() == built_for):
        return HOST_TARGET
    cuda = pathlib.Path(nvcc()).resolve().parent.parent
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DGDNR_BUILT_FOR="{built_for}"',
           "-I", str(root / "include"), "-I", str(root / "include" / "torch" / "csrc" / "api" / "include"),
           "-I", sysconfig.get_paths()["include"], "-I", str(cuda / "include"), str(HOST_SOURCE), "-o", str(HOST_TARGET),
           "-L", str(root / "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10_cuda", "-lc10"]
    print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    record.write_text(built_for)
    return HOST_TARGET


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose-ptxas", action="store_true")
    args = ap.parse_args()
    path = build(force=args.force, verbose_ptxas=args.verbose_ptxas)
    print(path)


if __name__ == "__main__":
    sys.exit(main())
