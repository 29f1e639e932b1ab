"""Builds the native libraries in-tree (they travel with the source tree).

    python -m malaga_b200.build

* libmalaga_b200.so — the CUDA engine (sm_100a only) behind include/malaga_b200.h
* libmgb_convert.so — host quantizers + seeded generator used by the converter
"""
from __future__ import annotations

import os
import re
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libmalaga_b200.so")
CONVERT_LIB = os.path.join(HERE, "libmgb_convert.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    # The arithmetic is specified op by op: no contraction of a*b+c into FMA
    # (explicit __fmaf_rn only), IEEE division and square root.
    "-fmad=false", "-prec-div=true", "-prec-sqrt=true",
    "-Xcompiler", "-fPIC,-fopenmp,-fvisibility=hidden",
    "-shared", "-lgomp",
    # device code of the many kernel instantiations is optimized in parallel
    "--split-compile=0",
]
# Compiled in one piece: with --split-compile the same source got one of several
# register assignments from build to build, which moved the attention kernels by up
# to 15 % and the logit rules from 29 to 33 us (34.5 in one piece; one row 6.9 us
# against 7.0 to 7.8). Level 3: the attention's tiles spill least and run fastest (8192
# tokens over 16384 keys of dim 128 in f16: 1.05 ms, 1.20 without; few rows take 1 to 3 %
# longer with it).
SOURCE_FLAGS = {"kvcache.cu": [], "kvattend.cu": ["-Xptxas=--register-usage-level=3"], "logits.cu": []}
ENGINE_SOURCES = ["engine.cu", "noalloc.cu", "kvcache.cu", "kvattend.cu", "logits.cu"]
OBJ_DIR = os.path.join(HERE, "_build")


def _newer(target: str, sources: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(s) > t for s in sources)


def _includes(path: str, seen: set[str] | None = None) -> set[str]:
    """`path` and every file that it includes by a quoted name, directly or not."""
    seen = set() if seen is None else seen
    path = os.path.realpath(path)
    if path not in seen and os.path.exists(path):
        seen.add(path)
        with open(path) as f:
            for name in re.findall(r'^\s*#include\s+"([^"]+)"', f.read(), re.M):
                _includes(os.path.join(os.path.dirname(path), name), seen)
    return seen


def build_lib(force: bool = False, verbose: bool = False) -> str:
    """Compiles the sources that are newer than their objects, side by side, and links them."""
    os.makedirs(OBJ_DIR, exist_ok=True)
    objects, running = [], []
    flags = [f for f in NVCC_FLAGS if f != "-shared"] + (["-Xptxas=-v"] if verbose else [])
    for name in ENGINE_SOURCES:
        src, obj = os.path.join(CSRC, name), os.path.join(OBJ_DIR, name + ".o")
        objects.append(obj)
        if force or _newer(obj, [*_includes(src), os.path.abspath(__file__)]):
            own = SOURCE_FLAGS.get(name)
            mine = flags if own is None else [f for f in flags if not f.startswith("--split-compile")] + own
            cmd = ["nvcc", *mine, "-c", src, "-o", obj + ".part"]
            running.append((cmd, obj, subprocess.Popen(cmd)))
    for cmd, obj, p in running:
        if p.wait() != 0:
            for _, _, other in running:
                other.wait()
            raise subprocess.CalledProcessError(p.returncode, cmd)
        os.replace(obj + ".part", obj)
    if force or _newer(LIB, objects):
        subprocess.check_call(["nvcc", *NVCC_FLAGS, *objects, "-o", LIB])
    return LIB


def build_convert(force: bool = False) -> str:
    src = os.path.join(CSRC, "convert", "quantize.cpp")
    if force or _newer(CONVERT_LIB, [src]):
        subprocess.check_call(["g++", "-O3", "-std=c++17", "-fopenmp", "-fPIC", "-shared", "-Wall", src,
                               "-o", CONVERT_LIB])
    return CONVERT_LIB


def build_all(force: bool = False) -> None:
    build_convert(force)
    build_lib(force)


if __name__ == "__main__":
    build_all(force="--force" in sys.argv)
