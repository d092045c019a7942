"""Build libgsec.so (the engine's C-ABI library) in-tree with nvcc for sm_100a.

    python 26mlsys-ae-ghostserve_b200/build.py [--force] [-v]

(and lib/gsec_torch.so, the calls of the KV-pool operators from torch tensors,
with g++ against torch's headers.)

Each ``csrc/*.cu`` compiles to an object under ``_build/`` (skipped when newer
than its sources and headers), then everything links into ``lib/libgsec.so``.
The CUDA runtime is linked statically so the library only needs the driver at
run time; it loads (but cannot launch) on a machine without a GPU.
"""
from __future__ import annotations

import concurrent.futures as cf
import glob
import importlib.metadata
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIBDIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIBDIR, "libgsec.so")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
CFLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-fvisibility=hidden",
          "-I", INCLUDE, "--expt-relaxed-constexpr"]


BIND = os.path.join(CSRC, "bind.cpp")
BIND_LIB = os.path.join(LIBDIR, "gsec_torch.so")
BIND_STAMP = os.path.join(BUILD, "gsec_torch.built_with")  # the torch and Python that BIND_LIB was built with


def _bind_versions() -> str:
    return f"torch {importlib.metadata.version('torch')}, {sysconfig.get_config_var('SOABI')}"


def _bind_stale() -> bool:
    """Whether BIND_LIB is missing, older than its sources, or built with another torch or Python."""
    if _stale(BIND_LIB, [BIND, *_headers()]) or not os.path.exists(BIND_STAMP):
        return True
    with open(BIND_STAMP) as f:
        return f.read() != _bind_versions()


def _build_bind(verbose: bool) -> None:
    """lib/gsec_torch.so: a Python module on top of libgsec.so (found beside it at run time)."""
    import torch
    from torch.utils import cpp_extension

    torch_lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    inc = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"], os.path.join(os.path.dirname(NVCC), "..", "include"),
           INCLUDE]
    cmd = ["g++", "-O2", "-std=c++20", "-fPIC", "-shared", "-fvisibility=hidden", "-Wno-deprecated",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *[f"-I{d}" for d in inc], BIND, "-o", BIND_LIB,
           f"-L{torch_lib}", f"-L{LIBDIR}", "-l:libgsec.so", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python",
           "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{torch_lib}"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for {BIND}:\n{r.stdout}\n{r.stderr}")
    with open(BIND_STAMP, "w") as f:
        f.write(_bind_versions())


def _headers():
    return glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h"))


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _compile(src, obj, verbose, ptxas_v):
    cmd = [NVCC, *ARCH, *CFLAGS, "-c", src, "-o", obj]
    if ptxas_v:
        cmd += ["-Xptxas", "-v"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    return r.stderr


def build(force: bool = False, verbose: bool = False, ptxas_v: bool = False) -> str:
    """Compile (if needed) and return the path of libgsec.so."""
    os.makedirs(BUILD, exist_ok=True)
    os.makedirs(LIBDIR, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    hdrs = _headers()
    jobs = []
    objs = []
    for src in srcs:
        obj = os.path.join(BUILD, os.path.basename(src)[:-3] + ".o")
        objs.append(obj)
        if force or ptxas_v or _stale(obj, [src, *hdrs]):
            jobs.append((src, obj))
    logs = []
    if jobs:
        with cf.ThreadPoolExecutor(max_workers=min(len(jobs), os.cpu_count() or 4)) as ex:
            for log in ex.map(lambda j: _compile(j[0], j[1], verbose, ptxas_v), jobs):
                logs.append(log)
    if ptxas_v:
        print("\n".join(logs))
    if force or jobs or _stale(LIB, objs):
        cmd = [NVCC, *ARCH, "-shared", "-o", LIB, *objs, "-cudart", "static"]
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    if force or _bind_stale():
        _build_bind(verbose)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv, ptxas_v="--ptxas" in sys.argv))
