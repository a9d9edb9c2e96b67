"""Builds libllmq.so (the sm_100a kernels and their C ABI) in this folder.

    python -m llm_mojo_b200.build

nvcc cross-compiles for sm_100a without a GPU. -fmad=false keeps each a*b+c
that the reference computes as two operations as two roundings; the kernels
call fmaf() where the reference calls .fma.
"""

from __future__ import annotations

import os
import re
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libllmq.so")
SOURCES = ["llmq.cu", "serving.cu", "quant_host.cpp"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def includes(path: str, seen: set[str] | None = None) -> set[str]:
    """path and the project's files that it includes, directly or not."""
    seen = set() if seen is None else seen
    if path not in seen:
        seen.add(path)
        with open(path) as f:
            for name in re.findall(r'^#include "(.+)"', f.read(), flags=re.M):
                includes(os.path.normpath(os.path.join(os.path.dirname(path), name)), seen)
    return seen


def stale(target: str, deps) -> bool:
    return not os.path.exists(target) or any(os.path.getmtime(d) > os.path.getmtime(target) for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compiles the sources that changed, side by side, and links them."""
    srcs = [os.path.join(CSRC, s) for s in SOURCES]
    if not force and not stale(LIB, set().union(*(includes(s) for s in srcs))):
        return LIB
    obj_dir = os.path.join(HERE, "_build")
    os.makedirs(obj_dir, exist_ok=True)
    objs, running = [], []
    for s in srcs:
        o = os.path.join(obj_dir, os.path.basename(s) + ".o")
        objs.append(o)
        if force or stale(o, includes(s)):
            cmd = [nvcc(), *ARCH, "-O3", "-lineinfo", "-std=c++17", "-fmad=false", "-Xcompiler",
                   "-fPIC,-ffp-contract=off,-O2", "-c", s, "-o", o]
            if verbose:
                print(" ".join(cmd))
            running.append((cmd, subprocess.Popen(cmd, cwd=CSRC)))
    for cmd, p in running:
        if p.wait():
            raise subprocess.CalledProcessError(p.returncode, cmd)
    cmd = [nvcc(), *ARCH, "-shared", "-o", LIB, *objs]
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True, cwd=CSRC)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
    print(LIB)
