"""Build libprism_bsa.so (sm_100a) in-tree with nvcc.

    python -m prism_b200.build          # or prism_b200.build.build()

Selection-side and correction-statistics sources are compiled with -fmad=false
(every floating-point step rounds once, in a fixed order); attention kernels use
default contraction.
"""
from __future__ import annotations

import contextlib
import fcntl
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


@contextlib.contextmanager
def _one_builder():
    """One process (and thread) of this machine builds at a time; the others find its files."""
    os.makedirs(BUILD, exist_ok=True)
    with open(os.path.join(BUILD, ".lock"), "w") as f:
        fcntl.flock(f, fcntl.LOCK_EX)
        yield


def _run(cmd, target: str, verbose: bool) -> None:
    """Runs a compiler whose output goes to ``target``, which appears there whole or not at all."""
    tmp = f"{target}.{os.getpid()}.tmp"
    cmd = cmd + ["-o", tmp]
    if verbose:
        print(" ".join(cmd), flush=True)
    try:
        subprocess.run(cmd, check=True)
        os.replace(tmp, target)
    finally:
        if os.path.exists(tmp):
            os.remove(tmp)


def build_torch_ops(verbose: bool = False, force: bool = False) -> str:
    with _one_builder():
        return _build_torch_ops(verbose, force)


def _build_torch_ops(verbose: bool, force: bool) -> str:
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
        cmd += [f"-I{d}" for d in includes] + [src, "-L" + os.path.join(base, "lib"), "-L" + HERE]
        # libprism_bsa.so is the one next to the extension; torch's libraries are loaded already
        cmd += ["-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda", "-lprism_bsa", "-Wl,-rpath,$ORIGIN"]
        _run(cmd, target, verbose)
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
    with _one_builder():
        return _build(verbose, force)


def _build(verbose: bool, force: bool) -> str:
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    headers.append(os.path.join(ROOT, "include", "prism_bsa.h"))
    objs = []
    for src, flags in SOURCES.items():
        s = os.path.join(CSRC, src)
        o = os.path.join(BUILD, src.replace(".cu", ".o"))
        objs.append(o)
        if force or _stale(o, [s] + headers):
            _run([nvcc()] + ARCH + COMMON + flags + ["-c", s], o, verbose)
    if force or _stale(LIB, objs):
        _run([nvcc()] + ARCH + ["-shared"] + objs, LIB, verbose)
    _build_torch_ops(verbose, force)
    return LIB


if __name__ == "__main__":
    build(verbose=True, force="--force" in sys.argv)
    print(LIB)
