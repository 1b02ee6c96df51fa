"""Build the sm_100a shared library in-tree, dolittle_b200/libdolittle_b200.so,
and the torch-side calls of dolittle_b200/shared.py, dolittle_b200/_torch_shared.*.so,
named after the Python and the torch that they were built for.

    python -m dolittle_b200.build [--verbose-ptxas]

Every kernel is compiled for sm_100a only (`-gencode arch=compute_100a,
code=sm_100a`) with --fmad=false: the reference compiles its CUDA sources the
same way, and the exact FP32 operation order of the parity kernels depends on
no implicit multiply-add contraction.  Objects go to dolittle_b200/_build/.
"""
from __future__ import annotations

import concurrent.futures as cf
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

from ._lib import torch_calls_path

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "libdolittle_b200.so")
TORCH_SRC = os.path.join(CSRC, "torch_shared.cpp")
BUILD = os.path.join(HERE, "_build")
ROOT = os.path.dirname(HERE)

NVCC = os.environ.get("NVCC", "nvcc")
CUDA_HOME = os.environ.get("CUDA_HOME", "/usr/local/cuda")
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "--fmad=false",
         "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
         "--expt-relaxed-constexpr", "-I", os.path.join(ROOT, "include")]


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def headers():
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh"))]
    hs.append(os.path.join(ROOT, "include", "dolittle_b200.h"))
    return hs


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build_torch_calls(force: bool = False):
    """The extension module that shared.py calls (host code only; torch's own
    libraries are already loaded when it is imported).  Returns its path, or
    None where it cannot be built: the C ABI and everything else do without it,
    and shared.py says what is missing."""
    header = os.path.join(ROOT, "include", "dolittle_b200.h")
    cxx, python = os.environ.get("CXX", "g++"), sysconfig.get_paths()["include"]
    try:
        out = torch_calls_path()
        root = os.path.dirname(importlib.util.find_spec("torch").origin)
    except ImportError:
        out = root = ""
    if out and not force and not _stale(out, [TORCH_SRC, header]):
        return out
    missing = [what for what, there in (
        ("torch", out),
        ("torch's headers", os.path.exists(os.path.join(root, "include", "ATen", "ATen.h"))),
        ("torch's CUDA library", os.path.exists(os.path.join(root, "lib", "libc10_cuda.so"))),
        ("Python's headers", os.path.exists(os.path.join(python, "Python.h"))),
        (cxx, shutil.which(cxx))) if not there]
    if missing:
        sys.stderr.write(f"dolittle_b200: the torch calls (dolittle_b200.shared) are not built: no {missing[0]}\n")
        return None
    import torch
    cmd = [cxx, "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", os.path.join(ROOT, "include"),
           "-I", os.path.join(root, "include"),
           "-I", os.path.join(root, "include", "torch", "csrc", "api", "include"),
           "-I", python, "-I", os.path.join(CUDA_HOME, "include"), TORCH_SRC,
           "-L", os.path.join(root, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python", "-o", out]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("torch calls failed to build:\n" + r.stdout + r.stderr)
    return out


def build(verbose_ptxas: bool = False, force: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    srcs = sources()
    hdrs = headers()
    jobs = []
    objs = []
    for s in srcs:
        o = os.path.join(BUILD, os.path.basename(s)[:-3] + ".o")
        objs.append(o)
        if force or _stale(o, [s] + hdrs):
            cmd = [NVCC, *FLAGS, "-c", s, "-o", o]
            if verbose_ptxas:
                cmd += ["-Xptxas", "-v"]
            jobs.append(cmd)

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        return cmd, r

    with cf.ThreadPoolExecutor(max_workers=min(8, max(1, len(jobs)))) as ex:
        for cmd, r in ex.map(run, jobs):
            if r.returncode != 0 or verbose_ptxas:
                sys.stderr.write(r.stdout + r.stderr)
            if r.returncode != 0:
                raise RuntimeError(f"nvcc failed: {' '.join(cmd)}")
    if force or jobs or _stale(OUT, objs):
        # NCCL (tensor-parallel all-reduce) is resolved with dlopen at run time.
        cmd = [NVCC, "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-o", OUT, *objs,
               "-lcudart", "-ldl"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("link failed:\n" + r.stdout + r.stderr)
    build_torch_calls(force)
    return OUT


if __name__ == "__main__":
    print(build(verbose_ptxas="--verbose-ptxas" in sys.argv, force="--force" in sys.argv))
