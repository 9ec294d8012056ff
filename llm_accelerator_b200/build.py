"""Builds libtaccel_b200.so (sm_100a) in-tree with nvcc, and behind it `_front`, the torch front ends' usual calls in C++.

The library holds the host compiler (instruction stream -> device plan), the
executor kernels and the stand-alone GEMM kernels.  It is built in the package
directory so it travels with the source tree; nothing is cached outside it.
`_front` speaks to torch's C++ side: its file is named by the torch and the
Python that it is built for, and without either's headers it is left out (the
front ends then make their calls in Python).
"""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
INCLUDE = PKG.parent / "include"
LIB = PKG / "libtaccel_b200.so"
OBJDIR = PKG.parent / "_build"
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
CXX = os.environ.get("CXX", "g++")
FRONT_SRC = CSRC / "tac_front.cc"
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", f"-I{INCLUDE}", f"-I{CSRC}"]


def sources() -> list[Path]:
    return sorted(list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cpp")))


def _deps() -> list[Path]:
    return sources() + sorted(CSRC.glob("*.h")) + sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))


def up_to_date() -> bool:
    if not LIB.exists():
        return False
    t = LIB.stat().st_mtime
    return all(p.stat().st_mtime <= t for p in _deps())


def front_path() -> Path:
    """The file of the extension module for this torch and this Python."""
    import torch
    abi = int(torch.compiled_with_cxx11_abi())
    return PKG / f"_front.torch-{torch.__version__}-abi{abi}{sysconfig.get_config_var('EXT_SUFFIX')}"


def front_missing() -> str | None:
    """Why the extension module cannot be built here, or None."""
    try:
        import torch
    except ImportError:
        return "torch is not installed"
    if torch.version.cuda is None:
        return "torch is built without CUDA"
    if not Path(sysconfig.get_path("include"), "Python.h").exists():
        return "Python's headers are not installed"
    return None


def front_up_to_date() -> bool:
    f = front_path()
    t = f.stat().st_mtime if f.exists() else 0
    return all(p.stat().st_mtime <= t for p in (FRONT_SRC, INCLUDE / "taccel_b200.h", _torch_dir() / "version.py"))


def _torch_dir() -> Path:
    import torch
    return Path(torch.__file__).resolve().parent


def build_front() -> Path:
    """Compile the extension module of the torch front ends, which calls the library by addresses."""
    import torch
    t, abi, front = _torch_dir(), int(torch.compiled_with_cxx11_abi()), front_path()
    tmp = front.with_name(front.name + ".tmp")
    cmd = [CXX, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={abi}", f"-I{INCLUDE}",
           *(f"-isystem{p}" for p in (t / "include", t / "include/torch/csrc/api/include", "/usr/local/cuda/include",
                                      sysconfig.get_path("include"))),
           str(FRONT_SRC), "-o", str(tmp), f"-L{t / 'lib'}", "-ltorch_python", "-ltorch_cuda", "-ltorch_cpu", "-lc10_cuda", "-lc10"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{CXX} failed for {FRONT_SRC.name}:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, front)
    return front


def _compile(src: Path, verbose: bool) -> Path:
    obj = OBJDIR / (src.name + ".o")
    cmd = [NVCC, *ARCH, *FLAGS, "-c", str(src), "-o", str(obj)]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{r.stdout}\n{r.stderr}")
    if verbose and r.stderr:
        sys.stderr.write(r.stderr)
    return obj


def build_library(force: bool = False, verbose: bool = False) -> Path:
    """Compile every CUDA / C++ source for sm_100a and link the shared library."""
    if not force and up_to_date():
        return LIB
    OBJDIR.mkdir(exist_ok=True)
    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose), sources()))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [NVCC, *ARCH, "-shared", "-o", str(tmp), *map(str, objs)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)
    return LIB


def build(force: bool = False, verbose: bool = False) -> Path:
    """The shared library, and then the front ends' module, where torch is there for it."""
    lib = build_library(force, verbose)
    if why := front_missing():
        sys.stderr.write(f"the torch front ends' module is left out: {why}\n")
    elif force or not front_up_to_date():
        build_front()
    return lib


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
