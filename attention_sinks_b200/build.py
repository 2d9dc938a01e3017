"""Builds the in-tree CUDA library `lib/libsinkcache_b200.so` with nvcc for sm_100a.

    python -m attention_sinks_b200.build [--force]

The library exports the C ABI declared in include/sinkcache_b200.h.  It links the CUDA
runtime statically, so it needs nothing at run time beyond the driver.
"""

import glob
import os
import re
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
SOURCES = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
# every header a translation unit may include: a change to one of them rebuilds the units that
# name it, and the library
HEADERS = sorted(glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h"))
                 + glob.glob(os.path.join(ROOT, "include", "*.h")))
LIB = os.path.join(HERE, "lib", "libsinkcache_b200.so")
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC,-O2",
]


def nvcc_path() -> str:
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the sm_100a CUDA library cannot be built")


def up_to_date() -> bool:
    if not os.path.exists(LIB):
        return False
    built = os.path.getmtime(LIB)
    return all(os.path.getmtime(p) <= built for p in SOURCES + HEADERS + [__file__])


def _included(path: str, seen: set[str] | None = None) -> set[str]:
    """`path` and every header of this tree that it includes, directly or not."""
    seen = set() if seen is None else seen
    path = os.path.realpath(path)
    if path not in seen and os.path.exists(path):
        seen.add(path)
        with open(path) as f:
            for name in re.findall(r'^\s*#include\s+"([^"]+)"', f.read(), flags=re.M):
                _included(os.path.join(os.path.dirname(path), name), seen)
    return seen


def _object(source: str, force: bool, verbose: bool) -> str:
    """The object file of one translation unit, compiled unless it is newer than all it includes."""
    obj = os.path.join(os.path.dirname(LIB), os.path.basename(source) + ".o")
    deps = [*_included(source), os.path.realpath(__file__)]
    if not force and os.path.exists(obj) and all(os.path.getmtime(p) <= os.path.getmtime(obj) for p in deps):
        return obj
    cmd = [nvcc_path(), *NVCC_FLAGS, "-c", source, "-o", obj + ".tmp"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(obj + ".tmp", obj)
    return obj


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile the library unless it is newer than every source; returns its path.  The
    translation units compile side by side."""
    if not force and up_to_date():
        return LIB
    os.makedirs(os.path.dirname(LIB), exist_ok=True)
    with ThreadPoolExecutor(len(SOURCES)) as pool:
        objects = list(pool.map(lambda src: _object(src, force, verbose), SOURCES))
    tmp = LIB + ".tmp"
    cmd = [nvcc_path(), "-shared", *NVCC_FLAGS, *objects, "-o", tmp]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
