"""Build libkvengine_b200.so in-tree for sm_100a (`python -m kvengine_b200.build`).

Plain nvcc invocations (no torch extension machinery): the library has a C ABI
and is loaded with ctypes. Objects go to `_build/` at the repository root.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
OBJDIR = os.path.join(ROOT, "_build")
LIB = os.path.join(PKG, "libkvengine_b200.so")
FAST = os.path.join(PKG, "_fastcall.so")  # the C++ binding of a sampling step's ops (csrc/fastcall.cpp)
SOURCES = ["capi.cu", "accept.cu", "kv.cu", "attention.cu", "gemm.cu", "gemm_simt.cu", "gemm_tc.cu",
           "forward.cu", "step.cu", "tree_attn.cu", "tree_attn_tc.cu", "tree_attn_small.cu",
           "kv_fp8.cu", "sample.cu", "kv_path.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ARCH + ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
                f"-I{INCLUDE}"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _newer(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return False
    t = os.path.getmtime(target)
    return all(os.path.getmtime(d) <= t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(OBJDIR, exist_ok=True)
    headers = [os.path.join(CSRC, h) for h in os.listdir(CSRC) if h.endswith((".cuh", ".h"))]
    headers.append(os.path.join(INCLUDE, "kvengine_b200.h"))
    cc = nvcc()
    jobs = []
    objs = []
    for src in SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(OBJDIR, src.replace(".cu", ".o"))
        objs.append(o)
        if force or not _newer(o, [s] + headers):
            jobs.append([cc] + FLAGS + ["-c", s, "-o", o])

    def run(cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
        return r

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        list(ex.map(run, jobs))
    if force or jobs or not _newer(LIB, objs):
        run([cc] + ARCH + ["-shared", "-o", LIB] + objs)
    build_fastcall(force, verbose)
    return LIB


def build_fastcall(force: bool = False, verbose: bool = False) -> str:
    """The CPython extension that calls the library from C++ (host code only; torch's headers)."""
    import sysconfig

    import torch

    src = os.path.join(CSRC, "fastcall.cpp")
    if not force and _newer(FAST, [src, os.path.join(INCLUDE, "kvengine_b200.h")]):
        return FAST
    if os.path.exists(FAST):  # one built for an older header would pass other arguments
        os.remove(FAST)
    home = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc())))
    cmd = [os.environ.get("CXX") or shutil.which("g++") or "c++", "-O2", "-std=c++17", "-fPIC", "-shared", "-w",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{home}/include",
           f"-I{home}/include/torch/csrc/api/include", f"-I{sysconfig.get_paths()['include']}", f"-I{cuda}/include", src,
           "-o", FAST, f"-L{home}/lib", "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"c++ failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    return FAST


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
