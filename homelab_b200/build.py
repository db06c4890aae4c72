"""Builds liboomb.so (the sm_100a kernels and their C ABI) in place.

    python -m homelab_b200.build

nvcc cross-compiles for sm_100a without a GPU.  The library lands next to
this file so it travels with the source tree.
"""
from __future__ import annotations

import os
import re
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
LIB = os.path.join(HERE, "liboomb.so")
SOURCES = [os.path.join(HERE, "csrc", f) for f in ("capi.cu", "paged.cu")]
OBJ_DIR = os.path.join(HERE, "build")
DEPS = [os.path.join(HERE, "csrc", f) for f in sorted(os.listdir(os.path.join(HERE, "csrc")))] + [
    os.path.join(ROOT, "include", "oomb.h")
]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "-Xptxas", "-v",
]


def nvcc() -> str:
    path = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(path):
        raise RuntimeError("nvcc not found: the sm_100a kernels cannot be built")
    return path


def stale(target: str = LIB, deps=None) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps or DEPS if os.path.exists(d))


def includes(path: str, seen=None) -> set:
    """`path` and the files it includes by a quoted name, transitively."""
    seen = set() if seen is None else seen
    path = os.path.realpath(path)
    if path not in seen and os.path.exists(path):
        seen.add(path)
        for name in re.findall(r'^\s*#include\s+"([^"]+)"', open(path).read(), re.M):
            includes(os.path.join(os.path.dirname(path), name), seen)
    return seen


def build(force: bool = False, verbose: bool = False) -> str:
    """Builds liboomb.so when a source is newer than it (or always with force): the
    translation units in parallel, each again only when a file it includes changed."""
    if not force and not stale():
        return LIB
    os.makedirs(OBJ_DIR, exist_ok=True)
    objs, jobs = [], []
    for src in SOURCES:
        obj = os.path.join(OBJ_DIR, os.path.basename(src) + ".o")
        objs.append(obj)
        if force or stale(obj, includes(src) | {os.path.realpath(__file__)}):
            cmd = [nvcc(), *NVCC_FLAGS, "-c", "-o", obj + ".tmp", src]
            jobs.append((obj, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    failed = False
    for obj, job in jobs:
        out, _ = job.communicate()
        if job.returncode != 0:
            failed = True
            sys.stderr.write(out)
        else:
            os.replace(obj + ".tmp", obj)
            if verbose:
                sys.stderr.write(out)
    if failed:
        raise RuntimeError("nvcc failed building liboomb.so")
    r = subprocess.run([nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-o", LIB + ".tmp", *objs],
                       capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("linking liboomb.so failed")
    os.replace(LIB + ".tmp", LIB)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
