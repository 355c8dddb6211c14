"""Build recipe for the sm_100a library (run from any directory).

    python 15-618_dynamic_sparse_decode_b200/build.py

produces, in this package directory:
    libdsd_b200.so        the C ABI (include/dsd_b200.h) + CUDA kernels
    libdsd_host.so        the drop-in C++ API (include/dsd/*.h) over the C ABI
    bin/dsd_bench, bin/dsd_continuous_bench   the drop-in CLIs
"""
from __future__ import annotations

import os
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
LIB = os.path.join(PKG, "libdsd_b200.so")

SOURCES = ["dsd_capi.cu", "dsd_scaled_capi.cu"]
HEADERS = ["dsd_internal.h", "dsd_kernels.cuh", "dsd_scaled_common.cuh", "dsd_scaled_append.cuh",
           "dsd_scaled_attn.cuh", "dsd_scaled_attn_tc.cuh", "dsd_scaled_attn_wide.cuh"]
# headers of one source only: the other need not be compiled again for them
ONLY = {"dsd_kernels.cuh": "dsd_capi.cu", "dsd_scaled_common.cuh": "dsd_scaled_capi.cu",
        "dsd_scaled_append.cuh": "dsd_scaled_capi.cu", "dsd_scaled_attn.cuh": "dsd_scaled_capi.cu",
        "dsd_scaled_attn_tc.cuh": "dsd_scaled_capi.cu",
        "dsd_scaled_attn_wide.cuh": "dsd_scaled_capi.cu"}


def _newer(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return False
    t = os.path.getmtime(target)
    return all(os.path.getmtime(d) <= t for d in deps)


def build_library(force: bool = False, verbose: bool = False, out: str = LIB,
                  defines: tuple = ()) -> str:
    """nvcc the C ABI + kernels into `out` (extra -D `defines` for experiments)."""
    flags = [*ARCH, "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC",
             *[f"-D{d}" for d in defines], f"-I{INCLUDE}", f"-I{CSRC}"]
    if verbose:
        flags.insert(0, "-Xptxas=-v")
    objects, jobs = [], []
    # objects of another library or with other defines lie beside it: never linked into this one
    at = os.path.join(PKG, "build") if out == LIB and not defines else os.path.abspath(out) + ".build"
    os.makedirs(at, exist_ok=True)
    for src in SOURCES:
        deps = [os.path.join(CSRC, src), os.path.join(INCLUDE, "dsd_b200.h")]
        deps += [os.path.join(CSRC, h) for h in HEADERS if ONLY.get(h, src) == src]
        obj = os.path.join(at, os.path.basename(out) + "." + src + ".o")
        objects.append(obj)
        if force or defines or not _newer(obj, deps):
            cmd = [NVCC, *flags, "-c", "-o", obj, os.path.join(CSRC, src)]
            if verbose:
                print(" ".join(cmd))
            jobs.append((cmd, subprocess.Popen(cmd)))
    for failed in [(job.returncode, cmd) for cmd, job in jobs if job.wait()]:   # all have ended by then
        raise subprocess.CalledProcessError(*failed)
    if jobs or not _newer(out, objects):
        subprocess.run([NVCC, *ARCH, "-shared", "-Xcompiler", "-fPIC", "-o", out, *objects], check=True)
    return out


HOST_DIR = os.path.join(CSRC, "host")
HOST_SOURCES = ["page_pool.cpp", "paged_kv_cache.cpp", "reference_kernels.cpp",
                "synthetic_data.cpp", "device_page_pool.cpp", "sparse_cuda_context.cpp",
                "decode_pipeline.cpp", "continuous_batching.cpp", "dense_stub.cpp"]
HOST_LIB = os.path.join(PKG, "libdsd_host.so")
BIN = os.path.join(PKG, "bin")
CLIS = {"dsd_bench": "bench_decode_main.cpp", "dsd_continuous_bench": "bench_continuous_main.cpp"}
CXX = os.environ.get("CXX", "g++")
# -ffp-contract=off: the CPU backends keep the reference's unfused arithmetic
CXXFLAGS = ["-O3", "-std=c++17", "-fPIC", "-ffp-contract=off", "-Wall", "-Wextra",
            f"-I{INCLUDE}", f"-I{HOST_DIR}"]


def build_host(force: bool = False) -> None:
    headers = [os.path.join(INCLUDE, "dsd", h) for h in os.listdir(os.path.join(INCLUDE, "dsd"))]
    headers += [os.path.join(HOST_DIR, h) for h in os.listdir(HOST_DIR) if h.endswith(".h")]
    headers += [os.path.join(INCLUDE, "dsd_b200.h")]
    srcs = [os.path.join(HOST_DIR, s) for s in HOST_SOURCES]
    if force or not _newer(HOST_LIB, srcs + headers + [LIB]):
        subprocess.run([CXX, *CXXFLAGS, "-shared", "-o", HOST_LIB, *srcs, f"-L{PKG}",
                        "-ldsd_b200", "-Wl,-rpath,$ORIGIN"], check=True)
    os.makedirs(BIN, exist_ok=True)
    for exe, src in CLIS.items():
        out = os.path.join(BIN, exe)
        s = os.path.join(HOST_DIR, src)
        if force or not _newer(out, [s, HOST_LIB] + headers):
            subprocess.run([CXX, *CXXFLAGS, "-o", out, s, f"-L{PKG}", "-ldsd_host", "-ldsd_b200",
                            "-Wl,-rpath,$ORIGIN/.."], check=True)


def build(force: bool = False, verbose: bool = False) -> None:
    build_library(force=force, verbose=verbose)
    build_host(force=force)


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
