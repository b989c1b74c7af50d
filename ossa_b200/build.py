"""Builds libossa_b200.so (the sm_100a kernels behind the C ABI) and _autograd.<abi>.so (the trainable
operators' autograd nodes, over that library and torch's) in-tree.

Run ``python -m ossa_b200.build`` or call :func:`build`.  Both are written next to this file so
that they travel with the source tree; nothing is installed into site-packages and no JIT cache is used.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

import torch

PKG_DIR = Path(__file__).resolve().parent
REPO_DIR = PKG_DIR.parent
CSRC = PKG_DIR / "csrc"
INCLUDE = REPO_DIR / "include"
LIB_NAME = "libossa_b200.so"
LIB_PATH = PKG_DIR / LIB_NAME
AUTOGRAD_SRC = CSRC / "autograd.cpp"


def _autograd_name() -> str:
    """The interpreter's and torch's versions are in the module's name: it is bound to the C++ ABI of both, and one
    built for others is not taken."""
    return f"_autograd.{sysconfig.get_config_var('SOABI')}.torch-{torch.__version__}.so"


AUTOGRAD_PATH = PKG_DIR / _autograd_name()

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [
    "-O3",
    "-std=c++17",
    "-lineinfo",
    "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC",
    "-Xcompiler", "-fvisibility=hidden",
]


def _nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found: the CUDA toolkit is required to build libossa_b200.so")
    return cand


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _inputs() -> list[Path]:
    return sources() + sorted(CSRC.glob("*.h")) + sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))


def autograd_is_stale() -> bool:
    if not AUTOGRAD_PATH.exists():
        return True
    built = AUTOGRAD_PATH.stat().st_mtime
    return any(p.stat().st_mtime > built for p in (AUTOGRAD_SRC, INCLUDE / "ossa_b200.h"))


def is_stale() -> bool:
    if not LIB_PATH.exists():
        return True
    built = LIB_PATH.stat().st_mtime
    return any(p.stat().st_mtime > built for p in _inputs())


def build_autograd(force: bool = False, verbose: bool = False) -> Path:
    """Compiles ``csrc/autograd.cpp`` against torch's headers and links the module to the library."""
    if not force and not autograd_is_stale():
        return AUTOGRAD_PATH
    torch_dir = Path(torch.__file__).resolve().parent
    inc, nvcc = torch_dir / "include", Path(_nvcc()).resolve()
    tmp = AUTOGRAD_PATH.with_suffix(f".{os.getpid()}.tmp")
    cmd = [shutil.which("g++") or "c++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", f"-I{INCLUDE}",
           "-isystem", str(inc), "-isystem", str(inc / "torch" / "csrc" / "api" / "include"),
           "-isystem", sysconfig.get_paths()["include"], "-isystem", str(nvcc.parent.parent / "include"),
           str(AUTOGRAD_SRC), "-o", str(tmp), f"-L{PKG_DIR}", "-lossa_b200", "-Wl,-rpath,$ORIGIN",
           f"-L{torch_dir / 'lib'}", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    res = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    if res.returncode != 0:
        raise RuntimeError("autograd.cpp failed:\n" + res.stdout.decode(errors="replace"))
    os.replace(tmp, AUTOGRAD_PATH)
    return AUTOGRAD_PATH


def build(force: bool = False, verbose: bool = False, jobs: int | None = None) -> Path:
    """Compiles every ``csrc/*.cu`` for sm_100a, links ``libossa_b200.so`` and builds the autograd module on it."""
    _build_library(force, verbose)
    build_autograd(force, verbose)
    return LIB_PATH


def _build_library(force: bool, verbose: bool) -> Path:
    if not force and not is_stale():
        return LIB_PATH
    nvcc = _nvcc()
    obj_dir = PKG_DIR / "_build"
    obj_dir.mkdir(exist_ok=True)
    objs = []
    procs = []
    for src in sources():
        obj = obj_dir / (src.stem + ".o")
        objs.append(obj)
        cmd = [nvcc, *ARCH_FLAGS, *NVCC_FLAGS, f"-I{INCLUDE}", f"-I{CSRC}", "-c", str(src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
    failed = []
    for src, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            failed.append((src, out.decode(errors="replace")))
        elif verbose and out:
            print(out.decode(errors="replace"), file=sys.stderr)
    if failed:
        msg = "\n".join(f"--- {s.name}\n{o}" for s, o in failed)
        raise RuntimeError(f"nvcc failed:\n{msg}")
    tmp = LIB_PATH.with_suffix(".so.tmp")
    link = [nvcc, *ARCH_FLAGS, "-shared", "-o", str(tmp), *map(str, objs)]
    if verbose:
        print(" ".join(link), file=sys.stderr)
    res = subprocess.run(link, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    if res.returncode != 0:
        raise RuntimeError("nvcc link failed:\n" + res.stdout.decode(errors="replace"))
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    force = "--force" in sys.argv
    print(build(force=force, verbose="-v" in sys.argv))
