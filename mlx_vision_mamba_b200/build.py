"""Builds libvmscan.so (the sm_100a selective-scan library) and _serving_ext.so
(the Python entry points of the serving operators) in-tree.

Usage: ``python -m mlx_vision_mamba_b200.build`` or ``build()`` from Python.
The library is a single nvcc translation unit (csrc/vmscan.cu) with the CUDA
runtime linked statically, so it loads without a GPU and travels with the
source tree.  The extension (csrc/serving_ext.cpp, g++) links against it and
against the installed PyTorch.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, "csrc")
LIB_PATH = os.path.join(PKG_DIR, "libvmscan.so")
SOURCES = ["vmscan.cu"]
DEPS = ["vmscan.cu", "vmscan_common.cuh", "vmscan_fwd.cuh", "vmscan_bwd.cuh", "vmscan_conv.cuh", "vmscan_dt.cuh",
        "vmscan_gemm.cuh", "vmscan_norm.cuh", "vmscan_cached.cuh", "vmscan_lora.cuh"]
EXT_PATH = os.path.join(PKG_DIR, "_serving_ext.so")
EXT_SOURCE = os.path.join(CSRC, "serving_ext.cpp")
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found: the CUDA toolkit is required to build libvmscan.so")
    return cand


def _stale() -> bool:
    if not os.path.exists(LIB_PATH):
        return True
    t = os.path.getmtime(LIB_PATH)
    root = os.path.dirname(PKG_DIR)
    deps = [os.path.join(CSRC, f) for f in DEPS] + [os.path.join(root, "include", "vmscan.h")]
    return any(os.path.getmtime(p) > t for p in deps if os.path.exists(p))


def build(force: bool = False, verbose: bool = False, extra_flags=None) -> str:
    """Compile libvmscan.so for sm_100a and _serving_ext.so if missing or out
    of date; return the library's path."""
    if force or _stale():
        _build_library(verbose, extra_flags)
    if force or _ext_stale():
        _build_ext()
    return LIB_PATH


def _build_library(verbose: bool, extra_flags) -> None:
    cmd = [
        nvcc_path(),
        *ARCH_FLAGS,
        "-O3",
        "-lineinfo",
        "-std=c++17",
        "-shared",
        "-Xcompiler",
        "-fPIC",
        "-cudart",
        "static",
        "-Xptxas",
        "-v" if verbose else "-O3",
        *(extra_flags or []),
        "-o",
        LIB_PATH + ".tmp",
        *[os.path.join(CSRC, s) for s in SOURCES],
    ]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + " ".join(cmd) + "\n" + proc.stdout + proc.stderr)
    if verbose:
        sys.stdout.write(proc.stdout + proc.stderr)
    os.replace(LIB_PATH + ".tmp", LIB_PATH)


def _ext_tag() -> str:
    """What the extension is tied to besides its sources: the installed PyTorch
    and the interpreter.  It is compiled in (serving_ext.cpp: kBuiltFor)."""
    import torch

    return f"serving_ext built for torch {torch.__version__} python {sys.version_info[0]}.{sys.version_info[1]};"


def _ext_stale() -> bool:
    if not os.path.exists(EXT_PATH):
        return True
    header = os.path.join(os.path.dirname(PKG_DIR), "include", "vmscan.h")
    if any(os.path.getmtime(p) > os.path.getmtime(EXT_PATH) for p in (EXT_SOURCE, header)):
        return True
    with open(EXT_PATH, "rb") as f:
        return _ext_tag().encode() not in f.read()


def _build_ext() -> None:
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    cuda_home = os.path.dirname(os.path.dirname(nvcc_path()))
    lib_dirs = [*cpp_extension.library_paths(), PKG_DIR]
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DVMSCAN_BUILT_FOR="{_ext_tag()}"']
    for inc in (*cpp_extension.include_paths(), sysconfig.get_paths()["include"], os.path.join(cuda_home, "include")):
        cmd += ["-isystem", inc]
    cmd += ["-o", EXT_PATH + ".tmp", EXT_SOURCE]
    for d in lib_dirs:
        cmd += ["-L" + d]
    cmd += ["-l:libvmscan.so", "-Wl,-rpath,$ORIGIN", "-ltorch_python", "-ltorch_cpu", "-ltorch", "-lc10_cuda", "-lc10", "-ldl"]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError("g++ failed:\n" + " ".join(cmd) + "\n" + proc.stdout + proc.stderr)
    os.replace(EXT_PATH + ".tmp", EXT_PATH)


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
