"""Build the in-tree C-ABI library ``aiwn_b200/libaiwn_il.so`` with nvcc.

    python aiwn_b200/csrc/build.py [--force]

(run as a file, so that building does not import -- and load -- the package)

Compiles every kernel for sm_100a only (``-gencode arch=compute_100a,
code=sm_100a``), with IEEE division and square root (no fast-math) so that
the bucketing is bit-exact with the reference.  cudart is linked statically,
so the library needs only the driver at run time.
"""
from __future__ import annotations

import glob
import os
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(HERE)
ROOT = os.path.dirname(PKG)
LIB = os.path.join(PKG, "libaiwn_il.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = [
    *ARCH,
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "-prec-div=true", "-prec-sqrt=true", "-ftz=false", "-fmad=true",
    "-Xptxas", "-warn-spills",
]


def sources():
    return units() + sorted(glob.glob(os.path.join(HERE, "*.cuh"))) + sorted(glob.glob(os.path.join(HERE, "*.h"))) + [
        os.path.join(ROOT, "include", "aiwn_il.h")]


def units():
    return sorted(glob.glob(os.path.join(HERE, "*.cu")))


def up_to_date() -> bool:
    if not os.path.exists(LIB):
        return False
    t = os.path.getmtime(LIB)
    return all(os.path.getmtime(s) <= t for s in sources())


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date():
        return LIB
    with tempfile.TemporaryDirectory() as tmp:
        objs = [os.path.join(tmp, os.path.basename(u) + ".o") for u in units()]
        cmds = [[NVCC, *FLAGS, "-I", os.path.join(ROOT, "include"), "-c", "-o", o, u] for o, u in zip(objs, units())]
        link = [NVCC, *ARCH, "--shared", "-cudart", "static", "-o", LIB + ".tmp", *objs]
        if verbose:
            print(*(" ".join(c) for c in (*cmds, link)), sep="\n")
        with ThreadPoolExecutor() as pool:  # the units are compiled side by side
            for _ in pool.map(lambda c: subprocess.run(c, check=True), cmds):
                pass
        subprocess.run(link, check=True)
    os.replace(LIB + ".tmp", LIB)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
