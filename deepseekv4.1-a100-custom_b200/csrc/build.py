"""Compile the CUDA sources of this package for sm_100a into one shared library, in-tree, and the Python extension that shortens the way to
the dense operators' forward calls.

    python deepseekv4.1-a100-custom_b200/csrc/build.py [--force] [--verbose]

Produces csrc/libb200moe.so and csrc/_fastcall.so (git-ignored).  nvcc cross-compiles without a GPU.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import glob
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(os.path.dirname(HERE))
LIB = os.path.join(HERE, "libb200moe.so")
FASTCALL = os.path.join(HERE, "_fastcall.so")
FASTCALL_KEY = os.path.join(HERE, "_obj", "fastcall.key")
NVCC = os.environ.get("B200MOE_NVCC", "nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
         "-I", os.path.join(ROOT, "include"), "-I", HERE]


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(HERE, "*.cu")))


def _deps() -> list[str]:
    return sources() + glob.glob(os.path.join(HERE, "*.cuh")) + glob.glob(os.path.join(ROOT, "include", "*.h")) + [os.path.abspath(__file__)]


def up_to_date() -> bool:
    if not os.path.exists(LIB):
        return False
    t = os.path.getmtime(LIB)
    return all(os.path.getmtime(d) <= t for d in _deps())


def _compile(src: str, verbose: bool) -> str:
    obj = os.path.join(HERE, "_obj", os.path.basename(src)[:-3] + ".o")
    cmd = [NVCC, *ARCH, *FLAGS, "-DB200_BUILDING=1", "-c", src, "-o", obj]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    if verbose:
        print(r.stderr)
    return obj


def fastcall_key() -> str:
    """What _fastcall.so is built against: it links torch's C++ interface, which another torch or Python does not share."""
    import torch
    return f"torch {torch.__version__}, python {sys.version.split()[0]}, cxx11 abi {int(torch.compiled_with_cxx11_abi())}\n"


def fastcall_up_to_date() -> bool:
    src = os.path.join(HERE, "fastcall.cpp")
    if not os.path.exists(FASTCALL) or not os.path.exists(FASTCALL_KEY):
        return False
    with open(FASTCALL_KEY) as f:
        return f.read() == fastcall_key() and all(os.path.getmtime(d) <= os.path.getmtime(FASTCALL) for d in (src, os.path.abspath(__file__)))


def build_fastcall(force: bool = False) -> str:
    """fastcall.cpp against the installed torch (host code only)."""
    if not force and fastcall_up_to_date():
        return FASTCALL
    import sysconfig

    import torch
    from torch.utils import cpp_extension as ext
    inc = [*ext.include_paths(), sysconfig.get_paths()["include"], os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")]
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", *(f for i in inc for f in ("-isystem", i)),
           os.path.join(HERE, "fastcall.cpp"), "-o", FASTCALL, *(f"-L{d}" for d in ext.library_paths()), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]
    if os.path.exists(FASTCALL_KEY):
        os.remove(FASTCALL_KEY)  # a build that is cut short leaves no key
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for fastcall.cpp:\n{r.stdout}\n{r.stderr}")
    os.makedirs(os.path.dirname(FASTCALL_KEY), exist_ok=True)
    with open(FASTCALL_KEY, "w") as f:
        f.write(fastcall_key())
    return FASTCALL


def build(force: bool = False, verbose: bool = False) -> str:
    with cf.ThreadPoolExecutor(max_workers=1) as side:  # beside nvcc
        fast = side.submit(build_fastcall, force)
        lib = build_library(force, verbose)
        fast.result()
    return lib


def build_library(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date():
        return LIB
    os.makedirs(os.path.join(HERE, "_obj"), exist_ok=True)
    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose), sources()))
    cmd = [NVCC, *ARCH, "-shared", "-o", LIB, *objs, "-lcudart_static", "-Xlinker", "--exclude-libs,ALL"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(a.force, a.verbose))
    sys.exit(0)
