"""Ahead-of-time build (in-tree, no JIT cache): libkore_b200.so with nvcc for sm_100a, and the Python module of the serving calls."""
from __future__ import annotations

import os
import shutil
import subprocess
import warnings

_PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(_PKG, "csrc")
LIB_DIR = os.path.join(_PKG, "_lib")
LIB_PATH = os.path.join(LIB_DIR, "libkore_b200.so")
SOURCES = ["api.cu", "quant.cu", "gemv.cu", "gemv_group.cu", "gemv_mma.cu", "gemv_stream.cu", "gemm_tc.cu", "gemm_tcs.cu", "gemm_tc2.cu", "static_scratch.cu", "shard.cu", "decoder_ops.cu", "decode_step.cu", "kv4.cu", "sample.cu"]
HEADERS = ["common.cuh", "device_utils.cuh", "tc_ptx.cuh", os.path.join("..", "..", "include", "kore_b200.h")]

MODULE_SOURCE = "serving_py.cpp"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC", "-shared",
    "-cudart", "static",
]


def nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found: the CUDA extension cannot be built")
    return exe


def stale() -> bool:
    if not os.path.exists(LIB_PATH):
        return True
    built = os.path.getmtime(LIB_PATH)
    deps = [os.path.join(CSRC, f) for f in SOURCES + HEADERS]
    return any(os.path.getmtime(d) > built for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile every CUDA source into one shared library, then the Python module; returns the library's path.  The library needs
    nvcc alone: where the module cannot be built (no torch headers, no C++ compiler) that is a warning."""
    if force or stale():
        os.makedirs(LIB_DIR, exist_ok=True)
        cmd = [nvcc(), *NVCC_FLAGS]
        if verbose:
            cmd += ["-Xptxas", "-v"]
        cmd += ["-o", LIB_PATH, *[os.path.join(CSRC, f) for f in SOURCES]]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError("nvcc failed:\n" + res.stdout + res.stderr)
        if verbose:
            print(res.stdout + res.stderr)
    try:
        build_module(force)
    except Exception as e:
        warnings.warn(f"the Python module of kore_b200.serving was not built: {e}", RuntimeWarning, stacklevel=2)
    return LIB_PATH


def module_path() -> str:
    """The Python module of kore_b200.serving, against torch's C++ headers; loads without a GPU.  Its name holds the Python and the
    torch that it is for: another one's is neither taken for current nor loaded."""
    import sysconfig

    import torch

    return os.path.join(LIB_DIR, f"kore_b200_serving.{sysconfig.get_config_var('SOABI')}.torch-{torch.__version__}.so")


def build_module(force: bool = False) -> str:
    """Compile the Python module of kore_b200.serving; returns its path."""
    import sysconfig

    import torch

    path = module_path()
    deps = [os.path.join(CSRC, MODULE_SOURCE), os.path.join(CSRC, HEADERS[-1])]
    if not force and os.path.exists(path) and all(os.path.getmtime(d) <= os.path.getmtime(path) for d in deps):
        return path
    os.makedirs(LIB_DIR, exist_ok=True)
    base = os.path.dirname(torch.__file__)
    includes = [os.path.join(base, "include"), os.path.join(base, "include", "torch", "csrc", "api", "include"),
                os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include"), sysconfig.get_paths()["include"]]
    cmd = [shutil.which("g++") or "c++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    for folder in includes:
        cmd += ["-isystem", folder]
    cmd += ["-o", path, deps[0], "-L" + os.path.join(base, "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("g++ failed:\n" + res.stdout + res.stderr)
    return path


if __name__ == "__main__":
    import sys

    print(build(force=True, verbose="-v" in sys.argv))
