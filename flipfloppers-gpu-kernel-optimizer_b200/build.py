"""Build libb200block.so in-tree with nvcc for sm_100a.

    python flipfloppers-gpu-kernel-optimizer_b200/build.py [--force] [--verbose]

The library is one translation unit (csrc/b200_block.cu includes every kernel
header) compiled with ``-gencode arch=compute_100a,code=sm_100a``.  Beside it,
``b200serving.so`` (csrc/serving_binding.cpp, host code only) is the Python
module of the serving operators' calls, linked to the library and to torch.  Both
land in ``lib/`` next to this file so they travel with the source tree.
"""

from __future__ import annotations

import argparse
import glob
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(REPO, "include")
LIB_DIR = os.path.join(HERE, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libb200block.so")
BINDING_SRC = os.path.join(CSRC, "serving_binding.cpp")
BINDING_PATH = os.path.join(LIB_DIR, "b200serving.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC,-O2", "-shared",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the CUDA 12.9 toolchain is required to build libb200block.so")


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh")) +
                  glob.glob(os.path.join(INCLUDE, "*.h")))


def up_to_date() -> bool:
    if not os.path.exists(LIB_PATH):
        return False
    t = os.path.getmtime(LIB_PATH)
    return all(os.path.getmtime(s) <= t for s in sources())


def build_binding(force: bool = False, verbose: bool = False) -> str:
    """The serving operators' Python module; needs the library built."""
    if not force and os.path.exists(BINDING_PATH) and all(
            os.path.getmtime(s) <= os.path.getmtime(BINDING_PATH)
            for s in (BINDING_SRC, os.path.join(INCLUDE, "b200_block.h"))):
        return BINDING_PATH
    import sysconfig

    import torch
    from torch.utils import cpp_extension as ext

    cxx = os.environ.get("CXX") or shutil.which("g++")
    if not cxx:
        raise RuntimeError("g++ not found: it is required to build b200serving.so")
    cuda = os.path.join(os.path.dirname(os.path.dirname(_nvcc())), "include")
    tmp = BINDING_PATH + ".tmp"
    cmd = [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-I", INCLUDE, "-I", sysconfig.get_paths()["include"], "-I", cuda]
    for d in ext.include_paths():
        cmd += ["-isystem", d]
    cmd += [BINDING_SRC, "-o", tmp, "-L", LIB_DIR, "-lb200block", "-Wl,-rpath,$ORIGIN"]
    for d in ext.library_paths():
        cmd += ["-L", d]
    cmd += ["-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, BINDING_PATH)
    return BINDING_PATH


def build(force: bool = False, verbose: bool = False, ptxas_info: bool = False) -> str:
    if not force and up_to_date():
        build_binding(verbose=verbose)
        return LIB_PATH
    os.makedirs(LIB_DIR, exist_ok=True)
    tmp = LIB_PATH + ".tmp"
    cmd = [_nvcc(), *NVCC_FLAGS, "-I", INCLUDE, "-I", CSRC, "-o", tmp, os.path.join(CSRC, "b200_block.cu")]
    if ptxas_info:
        cmd.insert(1, "-Xptxas=-v")
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
    if verbose or ptxas_info:
        sys.stdout.write(res.stdout + res.stderr)
    os.replace(tmp, LIB_PATH)
    build_binding(force=force, verbose=verbose)
    return LIB_PATH


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--ptxas-info", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose, ptxas_info=a.ptxas_info))
