"""Build libreels_lowvram.so in-tree for sm_100a (B200).

    python -m reels_b200.build [--force]

nvcc cross-compiles without a GPU; the .so is written next to this file so
it travels with the source tree.  Each .cu file is compiled on its own (in
parallel), and again only when it or a file it includes has changed.
"""
from __future__ import annotations

import glob
import os
import re
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "libreels_lowvram.so")
OBJ = os.path.join(HERE, "_build")

NVCC_FLAGS = [
    "-O3", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo",
    "-Xcompiler", "-fPIC", "-shared", "-Xptxas", "-warn-spills",
]


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))
                  + glob.glob(os.path.join(CSRC, "*.h"))
                  + glob.glob(os.path.join(ROOT, "include", "*.h")))


def _closure(path, seen=None):
    """The file and every file of the tree it includes, directly or not."""
    seen = set() if seen is None else seen
    path = os.path.normpath(path)
    if path not in seen and os.path.exists(path):
        seen.add(path)
        for name in re.findall(r'^\s*#include\s+"([^"]+)"', open(path).read(), re.M):
            _closure(os.path.join(os.path.dirname(path), name), seen)
    return seen


def _compile(src: str, force: bool, verbose: bool) -> str:
    obj = os.path.join(OBJ, os.path.basename(src)[:-3] + ".o")
    newest = max(os.path.getmtime(p) for p in _closure(src))
    if force or not os.path.exists(obj) or os.path.getmtime(obj) < newest:
        cmd = [os.environ.get("NVCC", "nvcc"), *(f for f in NVCC_FLAGS if f != "-shared"), "-c", "-o", obj, src]
        if verbose:
            print(" ".join(cmd))
        subprocess.run(cmd, check=True)
    return obj


def build(force: bool = False, verbose: bool = False) -> str:
    newest = max(os.path.getmtime(p) for p in sources())
    if not force and os.path.exists(OUT) and os.path.getmtime(OUT) >= newest:
        return OUT
    os.makedirs(OBJ, exist_ok=True)
    units = [p for p in sources() if p.endswith(".cu")]
    with ThreadPoolExecutor(len(units)) as pool:
        objects = list(pool.map(lambda p: _compile(p, force, verbose), units))
    cmd = [os.environ.get("NVCC", "nvcc"), "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-Xcompiler",
           "-fPIC", "-o", OUT, *objects]
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True)
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
