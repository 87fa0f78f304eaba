"""Build libhspmn_sm100.so, the sm_100a CUDA library behind hspmn_b200, and
libhspmn_torch.so, which registers its paged-cache operators with PyTorch.

Both are compiled in-tree (next to the Python package): the CUDA library with
nvcc for ``sm_100a`` only (the product has no other target), the operators
with the host compiler against the installed PyTorch. Each is rebuilt only
when a source it is made from is newer; the operators also when they were
built for another PyTorch or Python.

    python hspmn-v2.1_b200/build_native.py [--force] [-v]
"""

from __future__ import annotations

import argparse
import glob
import importlib.util
import os
import shutil
import subprocess
import sys
import warnings

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(REPO, "include")
LIB = os.path.join(HERE, "hspmn_b200", "libhspmn_sm100.so")
TORCH_LIB = os.path.join(HERE, "hspmn_b200", "libhspmn_torch.so")
TORCH_SOURCE = os.path.join(CSRC, "torch_ops.cpp")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "-shared", "-cudart", "static",
    "--expt-relaxed-constexpr",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; the HSPMN library needs the CUDA toolkit to build")


def cxx() -> str:
    """The system's host compiler. (A compiler that links its own libstdc++ in
    statically will not do: PyTorch's streams and the operators' must be one.)"""
    for cand in ("/usr/bin/g++", shutil.which("g++"), os.environ.get("CXX")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("g++ not found; the paged-cache operators need a host compiler to build")


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))
                  + glob.glob(os.path.join(INCLUDE, "*.h")))


def up_to_date(lib: str = LIB, made_from=None) -> bool:
    if not os.path.exists(lib):
        return False
    t = os.path.getmtime(lib)
    return all(os.path.getmtime(s) <= t for s in (made_from or sources()))


def run(cmd, out: str, verbose: bool) -> None:
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed:\n" + " ".join(cmd) + "\n" + r.stdout + r.stderr)
    if verbose:
        sys.stderr.write(r.stdout + r.stderr)
    os.replace(out + ".tmp", out)


def native():
    """The package's binding module, without the package."""
    spec = importlib.util.spec_from_file_location("hspmn_native", os.path.join(HERE, "hspmn_b200", "_native.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def torch_ops_up_to_date() -> bool:
    made_from = [TORCH_SOURCE, os.path.join(INCLUDE, "hspmn_sm100.h")]
    return up_to_date(TORCH_LIB, made_from) and native().built_for_this_torch(TORCH_LIB)


def build_torch_ops(force: bool = False, verbose: bool = False) -> str:
    if not force and torch_ops_up_to_date():
        return TORCH_LIB
    import sysconfig
    import torch
    from torch.utils.cpp_extension import include_paths, library_paths
    cuda_include = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc()))), "include")
    cmd = [cxx(), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DHSPMN_TORCH_BUILD_ID="{native().torch_build_id()}"',
           *(f"-isystem{p}" for p in (*include_paths(), cuda_include, sysconfig.get_paths()["include"])), "-I", INCLUDE, TORCH_SOURCE,
           "-o", TORCH_LIB + ".tmp", "-L", os.path.dirname(LIB), "-l:" + os.path.basename(LIB), "-Wl,-rpath,$ORIGIN",
           *(f"-L{p}" for p in library_paths()), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda",
           "-ltorch_python", "-ldl"]
    run(cmd, TORCH_LIB, verbose)
    with open(TORCH_LIB, "rb") as f:
        if b"libstdc++.so" not in f.read():
            os.remove(TORCH_LIB)
            raise RuntimeError(f"{cmd[0]} links libstdc++ statically; build with a compiler that uses the shared one")
    return TORCH_LIB


def build(force: bool = False, verbose: bool = False) -> str:
    if force or not up_to_date():
        cmd = [nvcc(), *NVCC_FLAGS, "-I", INCLUDE, "-I", CSRC,
               os.path.join(CSRC, "hspmn_sm100.cu"), "-o", LIB + ".tmp"]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        run(cmd, LIB, verbose)
    try:
        build_torch_ops(force, verbose)
    except (RuntimeError, ImportError, OSError) as e:
        # the C ABI and the other operators do not need it; calls of those that do raise
        warnings.warn(f"{os.path.basename(TORCH_LIB)} was not built, the paged-cache operators are missing: {e}",
                      RuntimeWarning, stacklevel=2)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose))
