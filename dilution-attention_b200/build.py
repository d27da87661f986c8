"""Build libdilution_b200.so in-tree with nvcc for sm_100a.

    python dilution-attention_b200/build.py [--force]

A translation unit is compiled again only when it or a file that it includes is newer than its
object.  nvcc cross-compiles without a GPU.
"""

from __future__ import annotations

import os
import re
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libdilution_b200.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xptxas=-v",
    "-Xcompiler", "-fPIC",
]
UNITS = ("abi.cu", "operators.cu", "trees.cu")     # one object each, next to its source


def _includes(path, seen=None):
    """The file and every file of this repository that it includes."""
    seen = set() if seen is None else seen
    path = os.path.normpath(path)
    if path in seen or not os.path.exists(path):
        return seen
    seen.add(path)
    with open(path) as f:
        for name in re.findall(r'^\s*#include "([^"]+)"', f.read(), re.M):
            _includes(os.path.join(os.path.dirname(path), name), seen)
    return seen


def _object(unit):
    return os.path.join(CSRC, unit.replace(".cu", ".o"))


def _stale(target, sources):
    return not os.path.exists(target) or any(os.path.getmtime(f) > os.path.getmtime(target) for f in sources)


def needs_build() -> bool:
    return any(_stale(LIB, _includes(os.path.join(CSRC, unit))) for unit in UNITS)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not needs_build():
        return LIB
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        raise RuntimeError("nvcc not found: cannot build libdilution_b200.so")

    def run(cmd):
        proc = subprocess.run(cmd, capture_output=True, text=True)
        if verbose or proc.returncode != 0:
            sys.stderr.write(proc.stdout + proc.stderr)
        return proc.returncode

    units = [u for u in UNITS if force or _stale(_object(u), _includes(os.path.join(CSRC, u)))]
    with ThreadPoolExecutor() as pool:
        codes = list(pool.map(lambda u: run([nvcc, *NVCC_FLAGS, "-c", "-o", _object(u), os.path.join(CSRC, u)]), units))
    if any(codes) or run([nvcc, *NVCC_FLAGS, "-shared", "-o", LIB, *map(_object, UNITS), "-lcuda"]):
        raise RuntimeError("nvcc failed building libdilution_b200.so")
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
