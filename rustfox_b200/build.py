"""Builds libfoxcuda.so in-tree with nvcc for sm_100a (no torch involved).

    python -m rustfox_b200.build [--verbose]
"""
from __future__ import annotations

import os
import re
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
SRCS = [os.path.join(HERE, "csrc", f) for f in ("foxcuda.cu", "kv4.cu")]
OBJ_DIR = os.path.join(HERE, "_build")
OUT = os.path.join(HERE, "libfoxcuda.so")
DEPS = [os.path.join(HERE, "csrc", f) for f in os.listdir(os.path.join(HERE, "csrc"))] + [
    os.path.join(HERE, "..", "include", "foxcuda.h")]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr", "-Xptxas", "-warn-spills",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    return "nvcc"


def up_to_date() -> bool:
    if not os.path.exists(OUT):
        return False
    t = os.path.getmtime(OUT)
    return all(os.path.getmtime(d) <= t for d in DEPS if os.path.exists(d))


def _includes(src: str) -> set:
    """src and the headers it includes by relative path, all the way down."""
    seen, todo = set(), [os.path.normpath(src)]
    while todo:
        f = todo.pop()
        if f in seen or not os.path.exists(f):
            continue
        seen.add(f)
        with open(f) as fh:
            todo += [os.path.normpath(os.path.join(os.path.dirname(f), m))
                     for m in re.findall(r'^\s*#include "([^"]+)"', fh.read(), flags=re.M)]
    return seen


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date():
        return OUT
    os.makedirs(OBJ_DIR, exist_ok=True)
    flags = [*NVCC_FLAGS, *(["-Xptxas", "-v"] if verbose else [])]
    jobs, objs = [], []
    for src in SRCS:  # one object per source, compiled side by side
        obj = os.path.join(OBJ_DIR, os.path.basename(src) + ".o")
        objs.append(obj)
        if force or not os.path.exists(obj) or any(os.path.getmtime(d) > os.path.getmtime(obj)
                                                     for d in _includes(src) | {__file__}):
            jobs.append((obj, subprocess.Popen([nvcc(), *flags, "-c", "-o", obj + ".tmp", src], text=True,
                                               stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
    failed = False
    for obj, job in jobs:
        log = job.communicate()[0]
        failed |= job.returncode != 0
        if job.returncode != 0 or verbose:
            sys.stderr.write(log)
        if job.returncode == 0:
            os.replace(obj + ".tmp", obj)
    if failed:
        raise RuntimeError("nvcc failed building libfoxcuda.so")
    # the CUDA runtime is linked statically: the library does not depend on
    # whichever libcudart another component of the process loaded
    res = subprocess.run([nvcc(), *NVCC_FLAGS, "-shared", "-cudart", "static", "-o", OUT + ".tmp", *objs],
                         capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("nvcc failed linking libfoxcuda.so")
    os.replace(OUT + ".tmp", OUT)
    return OUT


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="--verbose" in sys.argv)
    print(OUT)
