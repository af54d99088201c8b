"""Builds libqmlp_b200.so (host library + spec-independent kernels) in-tree with nvcc for sm_100a.

Usage: python quick-mlp_b200/build.py [--force]
The per-spec kernel instantiations are built on demand by the library itself (see csrc/jit.cpp) into
quick-mlp_b200/lib/specs/; `prebuild_specs` below instantiates a list of network specs ahead of time so a
machine without a compiler cache hit still finds them.
"""
import hashlib
import os
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIBDIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIBDIR, "libqmlp_b200.so")
SOURCES = ["host.cpp", "jit.cpp", "capi.cpp", "capi_operators.cpp", "generic_kernels.cu", "static_scratch.cu",
           "operators/common.cu", "operators/layer_norm.cu", "operators/embedding.cu", "operators/routing.cu", "operators/expert_linear.cu",
           "operators/dropout.cu", "operators/mx.cu", "operators/mx_linear.cu"]
NVCC = os.environ.get("QMLP_NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def _digest():
    h = hashlib.sha256()
    for root, _, files in sorted(os.walk(CSRC)):
        if os.path.basename(root) == "kernels":
            continue  # template headers only enter the per-spec instantiations
        for f in sorted(files):
            if f.endswith((".cpp", ".cu", ".cuh", ".h", ".hpp")):
                h.update(f.encode())
                h.update(open(os.path.join(root, f), "rb").read())
    h.update(open(os.path.join(CSRC, "kernels", "launch_args.h"), "rb").read())
    h.update(open(os.path.join(HERE, "..", "include", "qmlp_b200.h"), "rb").read())
    return h.hexdigest()


def build_library(force=False, verbose=True):
    os.makedirs(LIBDIR, exist_ok=True)
    stamp = os.path.join(LIBDIR, "libqmlp_b200.stamp")
    digest = _digest()
    if not force and os.path.exists(LIB) and os.path.exists(stamp) and open(stamp).read() == digest:
        return LIB
    flags = ["-std=c++17", "-O3", "-lineinfo", *ARCH, "-Xcompiler", "-fPIC,-fvisibility=hidden"]
    with tempfile.TemporaryDirectory() as objects:
        def compile_one(source):
            out = os.path.join(objects, source.replace("/", "_") + ".o")
            cmd = [NVCC, *flags, "-c", os.path.join(CSRC, source), "-o", out]
            if verbose:
                print(" ".join(cmd), flush=True)
            subprocess.check_call(cmd)
            return out
        with ThreadPoolExecutor(len(SOURCES)) as pool:
            linked = list(pool.map(compile_one, SOURCES))
        subprocess.check_call([NVCC, *flags, "-shared", "-o", LIB, *linked, "-ldl"])
    with open(stamp, "w") as f:
        f.write(digest)
    return LIB


if __name__ == "__main__":
    build_library(force="--force" in sys.argv)
    print("built", LIB)
