"""Build libprism_bsa.so (sm_100a) in-tree with nvcc.

    python -m prism_b200.build          # or prism_b200.build.build()

Selection-side and correction-statistics sources are compiled with -fmad=false
(every floating-point step rounds once, in a fixed order); attention kernels use
default contraction.
"""
from __future__ import annotations

import os
import re
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libprism_bsa.so")
ROOT = os.path.dirname(HERE)

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = ["-std=c++17", "-O3", "-lineinfo", "-Xcompiler", "-fPIC", "-I", os.path.join(ROOT, "include"),
          "--expt-relaxed-constexpr"]
SOURCES = {
    "select_kernels.cu": ["-fmad=false"],
    "correction_kernels.cu": ["-fmad=false"],
    "producer_kernels.cu": ["-fmad=false"],
    "bsa_tc.cu": [],
    "gemm_tc.cu": [],
    "gemm_fp8.cu": [],
    "norm_kernels.cu": [],
    "rotary_kernels.cu": [],
    "clip_kernels.cu": [],
}


def torch_ops_lib() -> str:
    """The extension of csrc/torch_ops.cpp, named after the torch and Python that it is built for."""
    import torch
    tag = f"{torch.__version__}_py{sys.version_info.major}{sys.version_info.minor}"
    return os.path.join(HERE, f"prism_torch_ops_{re.sub('[^0-9A-Za-z.]', '-', tag)}.so")


def build_torch_ops(verbose: bool = False, force: bool = False) -> str:
    import torch
    src, target = os.path.join(CSRC, "torch_ops.cpp"), torch_ops_lib()
    if force or _stale(target, [src, os.path.join(ROOT, "include", "prism_bsa.h")]):
        base = os.path.dirname(torch.__file__)
        cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc())))
        includes = [os.path.join(ROOT, "include"), os.path.join(base, "include"),
                    os.path.join(base, "include", "torch", "csrc", "api", "include"),
                    sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
        cmd = [shutil.which("g++") or "g++", "-std=c++17", "-O2", "-fPIC", "-shared",
               f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
        cmd += [f"-I{d}" for d in includes] + [src, "-o", target, "-L" + os.path.join(base, "lib"), "-L" + HERE]
        # libprism_bsa.so is the one next to the extension; torch's libraries are loaded already
        cmd += ["-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda", "-lprism_bsa", "-Wl,-rpath,$ORIGIN"]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
    return target


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _stale(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(verbose: bool = False, force: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    headers.append(os.path.join(ROOT, "include", "prism_bsa.h"))
    objs = []
    for src, flags in SOURCES.items():
        s = os.path.join(CSRC, src)
        o = os.path.join(BUILD, src.replace(".cu", ".o"))
        objs.append(o)
        if force or _stale(o, [s] + headers):
            cmd = [nvcc()] + ARCH + COMMON + flags + ["-c", s, "-o", o]
            if verbose:
                print(" ".join(cmd), flush=True)
            subprocess.run(cmd, check=True)
    if force or _stale(LIB, objs):
        cmd = [nvcc()] + ARCH + ["-shared", "-o", LIB] + objs
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
    build_torch_ops(verbose=verbose, force=force)
    return LIB


if __name__ == "__main__":
    build(verbose=True, force="--force" in sys.argv)
    print(LIB)
