"""Build the in-tree CUDA library ``libqrb200.so`` for sm_100a with nvcc, and its Python binding.

The library exposes only the C ABI declared in ``include/qrb200.h`` (no torch types), so it
is compiled directly with nvcc rather than through a torch extension. ``_native.so`` is the
native binding of the operators on 8- and 4-bit data: host code only, compiled against torch's
headers and linked to the library beside it. Run as
``python -m qr_v2_b200_kernel_b200.build`` or call :func:`build`.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_DIR = os.path.dirname(PKG_DIR)
CSRC = os.path.join(PKG_DIR, "csrc")
LIB_NAME = "libqrb200.so"
LIB_PATH = os.path.join(PKG_DIR, LIB_NAME)
SOURCES = ["qrb200.cu", "quant.cu", "fp8.cu", "kv8.cu", "noalloc.cu"]
NATIVE_PATH = os.path.join(PKG_DIR, "_native.so")
NATIVE_SOURCE = os.path.join(CSRC, "native.cpp")
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; the qrb200 CUDA library cannot be built")


def _inputs() -> list[str]:
    files = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh", ".h"))]
    files.append(os.path.join(REPO_DIR, "include", "qrb200.h"))
    return files


def _newer(target: str, inputs: list[str]) -> bool:
    if not os.path.exists(target):
        return False
    t = os.path.getmtime(target)
    return all(os.path.getmtime(f) <= t for f in inputs)


def up_to_date() -> bool:
    return _newer(LIB_PATH, _inputs()) and _native_up_to_date()


def _native_up_to_date() -> bool:
    return _newer(NATIVE_PATH, [NATIVE_SOURCE, os.path.join(REPO_DIR, "include", "qrb200.h")])


def _native_command() -> list[str]:
    """g++ on the binding, against the headers and libraries of the torch that is installed."""
    import sysconfig

    import torch

    root = os.path.dirname(torch.__file__)
    include, lib = os.path.join(root, "include"), os.path.join(root, "lib")
    cuda = os.path.dirname(os.path.dirname(nvcc_path()))
    return ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
            "-I", os.path.join(REPO_DIR, "include"), "-I", include,
            "-I", os.path.join(include, "torch", "csrc", "api", "include"), "-I", os.path.join(cuda, "include"),
            "-I", sysconfig.get_paths()["include"], NATIVE_SOURCE, "-o", NATIVE_PATH + ".tmp", LIB_PATH, "-L", lib,
            "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python",
            "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{lib}"]


def _run(cmd: list[str], what: str) -> str:
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{what} failed ({res.returncode}):\n{res.stderr}\n{res.stdout}")
    return res.stderr


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile ``libqrb200.so`` and ``_native.so`` next to this file where a source is newer; return the library's path."""
    if force or not _newer(LIB_PATH, _inputs()):
        # Without -soname the binding would record the path it was linked with.
        cmd = [nvcc_path(), *ARCH_FLAGS, "-O3", "-lineinfo", "-std=c++17", "-shared", "--threads", "0",
               "-Xcompiler", "-fPIC", "-Xlinker", f"-soname={LIB_NAME}", "-Xptxas", "-v" if verbose else "-O3",
               "-I", os.path.join(REPO_DIR, "include"), "-o", LIB_PATH + ".tmp"]
        cmd += [os.path.join(CSRC, s) for s in SOURCES]
        log = _run(cmd, "nvcc")
        if verbose:
            sys.stderr.write(log)
        os.replace(LIB_PATH + ".tmp", LIB_PATH)
    if force or not _native_up_to_date():
        _run(_native_command(), "g++")
        os.replace(NATIVE_PATH + ".tmp", NATIVE_PATH)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
