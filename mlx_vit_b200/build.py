"""Build libkda_b200.so in-tree with nvcc for sm_100a (B200).

``python -m mlx_vit_b200.build`` (or ``__graft_entry__.build()``) compiles every ``.cu``
under ``mlx_vit_b200/csrc`` into ``mlx_vit_b200/libkda_b200.so``.  Objects go to
``mlx_vit_b200/_build`` and are rebuilt when a source or header is newer.  The host module
``mlx_vit_b200/_tensors.so`` (csrc/tensors_module.cpp, against torch's headers) is built with g++.
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
OUT = os.path.join(PKG, "libkda_b200.so")
HOST_SRC, HOST_OUT = os.path.join(CSRC, "tensors_module.cpp"), os.path.join(PKG, "_tensors.so")
BUILD = os.path.join(PKG, "_build")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "--use_fast_math", "-Xcompiler", "-fPIC",
         "-Xcompiler", "-fvisibility=hidden", "--expt-relaxed-constexpr"]
# sources whose results are defined by separately rounded float32 operations
EXACT = {"kda_adamw.cu"}


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _deps():
    return glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(ROOT, "include", "*.h"))


def build_host(verbose: bool = False) -> str:
    """The CPython module around the library's host-bound operators."""
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths, library_paths
    newest = max([os.path.getmtime(HOST_SRC)] + [os.path.getmtime(p) for p in _deps()])
    if os.path.exists(HOST_OUT) and os.path.getmtime(HOST_OUT) >= newest:
        return HOST_OUT
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-isystem", sysconfig.get_paths()["include"], *(f for p in include_paths() for f in ("-isystem", p)),
           "-isystem", os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include"),
           HOST_SRC, "-o", HOST_OUT, *(f"-L{p}" for p in library_paths()), f"-L{PKG}", "-Wl,-rpath,$ORIGIN",
           "-l:libkda_b200.so", "-ltorch_python", "-ltorch_cpu", "-lc10_cuda", "-lc10"]
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True)
    return HOST_OUT


def build(verbose: bool = False, extra_flags=()) -> str:
    os.makedirs(BUILD, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    hdr_mtime = max([os.path.getmtime(p) for p in _deps()] + [0])
    objs = []
    for src in srcs:
        obj = os.path.join(BUILD, os.path.basename(src) + ".o")
        objs.append(obj)
        if os.path.exists(obj) and os.path.getmtime(obj) >= max(os.path.getmtime(src), hdr_mtime):
            continue
        flags = [f for f in FLAGS if f != "--use_fast_math" or os.path.basename(src) not in EXACT]
        cmd = [nvcc(), *ARCH, *flags, *extra_flags, "-I", os.path.join(ROOT, "include"),
               "-c", src, "-o", obj]
        if verbose:
            print(" ".join(cmd))
        subprocess.run(cmd, check=True)
    if not os.path.exists(OUT) or os.path.getmtime(OUT) < max(os.path.getmtime(o) for o in objs):
        cmd = [nvcc(), *ARCH, "-shared", "-Xcompiler", "-fPIC", *objs, "-o", OUT, "-lcudart"]
        subprocess.run(cmd, check=True)
    build_host(verbose)
    return OUT


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
