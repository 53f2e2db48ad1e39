"""Build recipe for libbitcache_b200.so (sm_100a), in-tree.

Each CUDA source under csrc/ is compiled with nvcc for sm_100a only and linked
into ``bitcache_b200/libbitcache_b200.so`` next to this file.  The flags match
the reference build (``-O3 --use_fast_math``): the encoders rely on the same
fast-math division as the reference kernels to produce bit-identical INT4
codes and scales.  Sources in IEEE_SOURCES are compiled without fast-math and
without contraction: their results are defined by correctly rounded operations.

Usage: ``python -m bitcache_b200.build`` (rebuilds what changed).
"""
from __future__ import annotations

import concurrent.futures as cf
import glob
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(ROOT, "include")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libbitcache_b200.so")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-I", INCLUDE, "-I", CSRC]
IEEE_SOURCES = ("rope.cu",)


def nvcc() -> str:
    return os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")


def _deps() -> list[str]:
    return [f for d in (CSRC, INCLUDE) for end in ("*.h", "*.cuh") for f in glob.glob(os.path.join(d, end))] + [__file__]


def _stale(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _compile(src: str, extra: list[str]) -> str:
    obj = os.path.join(BUILD, os.path.basename(src) + ".o")
    if _stale(obj, [src] + _deps()):
        fast = ["-fmad=false"] if os.path.basename(src) in IEEE_SOURCES else ["--use_fast_math"]
        cmd = [nvcc(), *ARCH, *NVCC_FLAGS, *fast, *extra, "-c", src, "-o", obj]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed for {src}:\n{r.stderr}")
    return obj


def build(verbose_ptxas: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    extra = ["-Xptxas", "-v"] if verbose_ptxas else []
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        objs = list(ex.map(lambda s: _compile(s, extra), srcs))
    if _stale(LIB, objs):
        cmd = [nvcc(), *ARCH, "-shared", "-Xcompiler", "-fPIC", *objs, "-o", LIB + ".tmp", "-lcudart"]
        subprocess.run(cmd, check=True)
        os.replace(LIB + ".tmp", LIB)
    return LIB


if __name__ == "__main__":
    print(build(verbose_ptxas="-v" in sys.argv))
