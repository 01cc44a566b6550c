"""Build recipe for the in-tree CUDA library (libqdecode.so, sm_100a).

The library is compiled with nvcc directly (no torch extension machinery): it is
a plain C-ABI shared object that JavaScript, C or Python can load. Beside it, for the
installed torch, _torch_calls.so: the Python module through which runtime.py's paged
operators and batched sampler take torch tensors (csrc/torch_calls.cpp). It is built apart
(build_calls), when one of them is first called: nothing else needs it.
"""
from __future__ import annotations

import hashlib
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
LIB = os.path.join(PKG, "libqdecode.so")
SOURCES = ["engine.cu", "batch.cu", "noalloc.cu", "bench_api.cu", "sample.cu", "paged.cu", "sample_rows.cu",
           "score_rows.cu"]
DEPS = SOURCES + ["kernels.cuh", "persist.cuh", "gemm_tc.cuh", "batch.cuh", "paged.cuh", "paged_decode.cuh", "paged_prompt.cuh", "paged_q8.cuh", "paged_shared.cuh", "rows.cuh", "internal.cuh", "overlap.hpp", "tma.cuh", "common.cuh", "json.hpp"]
CALLS = os.path.join(PKG, "_torch_calls.so")
CALLS_SOURCE = "torch_calls.cpp"
CALLS_KEY = os.path.join(PKG, "_build", "torch_calls.key")  # what the module on disk was built from
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    paths = [os.path.join(CSRC, d) for d in DEPS] + [os.path.join(ROOT, "include", "qdecode.h")]
    return any(os.path.getmtime(p) > t for p in paths)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not _stale():
        return LIB
    obj_dir = os.path.join(PKG, "_build")
    os.makedirs(obj_dir, exist_ok=True)
    common = [nvcc(), "-O3", "-std=c++17", *ARCH, "-lineinfo", "-Xcompiler", "-fPIC,-O3",
              "-I", os.path.join(ROOT, "include")]
    if verbose:
        common += ["-Xptxas", "-v"]
    # one nvcc per translation unit, in parallel, then one link
    procs, objs = [], []
    for src in SOURCES:
        obj = os.path.join(obj_dir, src.replace(".cu", ".o"))
        objs.append(obj)
        procs.append((src, subprocess.Popen(common + ["-c", os.path.join(CSRC, src), "-o", obj],
                                            stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)))
    failed = False
    for src, p in procs:
        out, err = p.communicate()
        if p.returncode != 0:
            sys.stderr.write(f"--- {src}\n" + out + err)
            failed = True
        elif verbose:
            sys.stderr.write(err)
    if failed:
        raise RuntimeError("nvcc failed building libqdecode.so")
    res = subprocess.run([nvcc(), *ARCH, "-shared", "-o", LIB + ".tmp", *objs], capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("nvcc failed linking libqdecode.so")
    os.replace(LIB + ".tmp", LIB)
    return LIB


def _calls_key(torch) -> str:
    """The torch and Python that a module built now belongs to, and its sources."""
    h = hashlib.sha256()
    for path in (os.path.join(CSRC, CALLS_SOURCE), os.path.join(CSRC, "overlap.hpp"), os.path.join(ROOT, "include", "qdecode.h")):
        with open(path, "rb") as f:
            h.update(f.read())
    return f"torch {torch.__version__} {sys.implementation.cache_tag} {h.hexdigest()}"


def build_calls(force: bool = False) -> str:
    """_torch_calls.so against the installed torch and libqdecode.so ("" where there is no torch)."""
    if importlib.util.find_spec("torch") is None:
        return ""
    import torch
    key = _calls_key(torch)
    if not force and os.path.exists(CALLS) and os.path.exists(CALLS_KEY):
        with open(CALLS_KEY) as f:
            if f.read() == key:
                return CALLS
    home = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(nvcc()))
    mine = f".{os.getpid()}.tmp"  # processes may build at once
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", os.path.join(CSRC, CALLS_SOURCE), "-o", CALLS + mine,
           "-I", os.path.join(home, "include"), "-I", os.path.join(home, "include", "torch", "csrc", "api", "include"),
           "-I", sysconfig.get_paths()["include"], "-I", os.path.join(cuda, "include"), "-L", os.path.join(home, "lib"),
           "-ltorch_python", "-ltorch_cpu", "-ltorch", "-lc10", "-lc10_cuda", "-L", PKG, "-lqdecode", "-Wl,-rpath,$ORIGIN"]
    try:
        res = subprocess.run(cmd, capture_output=True, text=True)
    except OSError as err:
        raise RuntimeError(f"no g++ to build _torch_calls.so with: {err}") from err
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("g++ failed building _torch_calls.so")
    os.replace(CALLS + mine, CALLS)
    os.makedirs(os.path.dirname(CALLS_KEY), exist_ok=True)
    with open(CALLS_KEY + mine, "w") as f:
        f.write(key)
    os.replace(CALLS_KEY + mine, CALLS_KEY)
    return CALLS


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    build_calls(force="--force" in sys.argv)
    print(LIB)
