"""Builds liblucid_cuda.so (sm_100a) next to this file with nvcc, and two small CPython modules that spare
eager calls the host time of ctypes and Python: ``_fastcall`` (gcc, no dependency) binds a few entry points,
``_torchcall`` (g++ against torch's headers) checks and allocates for the functional operators.

    python -m lucid_b200._C.build [--force]

nvcc cross-compiles without a GPU.  The shared object is kept in-tree so that it
travels with the source tree; it is not installed into site-packages.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(os.path.dirname(HERE))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(ROOT, "include")
OBJ_DIR = os.path.join(HERE, "build")
LIB_PATH = os.path.join(HERE, "liblucid_cuda.so")
FASTCALL_SRC = os.path.join(CSRC, "fastcall.c")
FASTCALL_PATH = os.path.join(HERE, "_fastcall" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))

TORCHCALL_SRC = os.path.join(CSRC, "torchcall.cpp")
TORCHCALL_PATH = os.path.join(HERE, "_torchcall" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))

SOURCES = ["api.cu", "quant_kernels.cu", "hist_kernels.cu", "embed_kernels.cu", "qlinear_tcgen05.cu", "wo_kernels.cu",
           "wo_prep_kernels.cu", "peer_kernels.cu", "qgemv_kernels.cu", "grouped_tcgen05.cu", "expert_kernels.cu"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "-I", INCLUDE, "-I", CSRC,
]


def _nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found; liblucid_cuda.so cannot be built")
    return exe


def _newer(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return False
    t = os.path.getmtime(target)
    return all(os.path.getmtime(d) <= t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile every .cu and link the shared library; returns its path."""
    os.makedirs(OBJ_DIR, exist_ok=True)
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    headers.append(os.path.join(INCLUDE, "lucid_cuda.h"))
    nvcc = _nvcc()
    objs, jobs = [], []
    for src in SOURCES:
        src_path = os.path.join(CSRC, src)
        obj = os.path.join(OBJ_DIR, src.replace(".cu", ".o"))
        objs.append(obj)
        if force or not _newer(obj, [src_path] + headers):
            jobs.append([nvcc, *NVCC_FLAGS, "-c", src_path, "-o", obj])

    def run(cmd: list[str]) -> None:
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"compiler failed:\n{' '.join(cmd)}\n{r.stdout}\n{r.stderr}")

    with ThreadPoolExecutor(max_workers=4) as pool:
        list(pool.map(run, jobs))
    if force or jobs or not _newer(LIB_PATH, objs):
        run([nvcc, "-shared", "-o", LIB_PATH, *objs, "-gencode", "arch=compute_100a,code=sm_100a"])
    if force or not _newer(FASTCALL_PATH, [FASTCALL_SRC, os.path.join(INCLUDE, "lucid_cuda.h")]):
        cc = shutil.which("gcc") or shutil.which("cc")
        if cc is None:
            raise RuntimeError("gcc not found; the _fastcall module cannot be built")
        run([cc, "-O2", "-shared", "-fPIC", "-Wall", "-I", sysconfig.get_paths()["include"], "-I", INCLUDE,
             FASTCALL_SRC, "-o", FASTCALL_PATH])
    if force or not _newer(TORCHCALL_PATH, [TORCHCALL_SRC, os.path.join(INCLUDE, "lucid_cuda.h")]):
        import torch
        from torch.utils import cpp_extension

        cxx = shutil.which("g++") or shutil.which("c++")
        if cxx is None:
            raise RuntimeError("g++ not found; the _torchcall module cannot be built")
        lib_dir = os.path.join(os.path.dirname(torch.__file__), "lib")
        cuda_include = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc))), "include")
        run([cxx, "-O2", "-std=c++17", "-shared", "-fPIC", "-Wall",
             f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", sysconfig.get_paths()["include"],
             *[f"-isystem{d}" for d in cpp_extension.include_paths()], f"-isystem{cuda_include}", "-I", INCLUDE,
             TORCHCALL_SRC, "-o", TORCHCALL_PATH, "-L", lib_dir, "-lc10", "-lc10_cuda", "-ltorch_cpu",
             "-ltorch_python"])
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
