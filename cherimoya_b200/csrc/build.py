"""Build libcherimoya_b200.so (sm_100a) in-tree with nvcc.

    python -m cherimoya_b200.csrc.build [--verbose]

The library is plain CUDA C++ behind the C ABI of include/cherimoya_b200.h
(no torch headers), so it builds in seconds and loads with ctypes.
"""

import os
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(HERE)
ROOT = os.path.dirname(PKG)
LIB = os.path.join(PKG, "libcherimoya_b200.so")
SOURCES = [os.path.join(HERE, f) for f in (
    "chm_engine.cu", "chm_likelihood.cu", "chm_likelihood_f32.cu", "chm_likelihood_bf16.cu",
    "chm_likelihood_f16.cu")]
DEPS = SOURCES + [os.path.join(HERE, f) for f in (
    "chm_kernels.cuh", "chm_likelihood.cuh", "chm_likelihood_run.cuh", "chm_likelihood.h",
    "chm_exp64.h", "chm_host.h", "chm_ptx.cuh")] + [
    os.path.join(ROOT, "include", "cherimoya_b200.h")]


def nvcc_path():
    cand = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
    return cand if os.path.exists(cand) else "nvcc"


def needs_build():
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    return any(os.path.getmtime(d) > t for d in DEPS)


def build(verbose=False, force=False):
    if not force and not needs_build():
        return LIB
    arch = ["-gencode", "arch=compute_100a,code=sm_100a"]
    flags = arch + ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-O2"]
    if verbose:
        flags += ["-Xptxas", "-v"]
    with tempfile.TemporaryDirectory() as tmp:
        objs = [os.path.join(tmp, os.path.basename(src) + ".o") for src in SOURCES]
        # one compiler per source, side by side
        with ThreadPoolExecutor(len(SOURCES)) as pool:
            done = list(pool.map(lambda a: _nvcc(flags + ["-c", a[0], "-o", a[1]]),
                                 zip(SOURCES, objs)))
        log = "".join(done) + _nvcc(arch + ["-shared", "-o", LIB + ".tmp"] + objs)
    if verbose:
        sys.stderr.write(log)
    os.replace(LIB + ".tmp", LIB)
    return LIB


def _nvcc(args):
    res = subprocess.run([nvcc_path()] + args, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("nvcc failed building libcherimoya_b200.so")
    return res.stderr


if __name__ == "__main__":
    build(verbose="--verbose" in sys.argv, force=True)
    print(LIB)
