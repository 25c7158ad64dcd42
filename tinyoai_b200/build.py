"""Builds libtinyoai_cuda.so in-tree with nvcc for sm_100a.

Two sources carry the C ABI of include/tinyoai_cuda.h: csrc/runtime.cu (models
and sessions) and csrc/paged.cu (operators over a caller's paged cache). They
compile side by side; an object is rebuilt when a file it includes is newer.
nvcc cross-compiles without a GPU.
"""
import os
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
LIB = PKG / "libtinyoai_cuda.so"
OBJ_DIR = PKG / "_build"
SOURCES = [PKG / "csrc" / "runtime.cu", PKG / "csrc" / "paged.cu"]
DEPS = sorted((PKG / "csrc").glob("*.cu*")) + sorted((PKG / "csrc").glob("*.h")) + [ROOT / "include" / "tinyoai_cuda.h"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "-Xcudafe", "--diag_suppress=177",
]


def nvcc():
    for cand in [os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"]:
        if cand and (os.path.isabs(cand) and os.path.exists(cand) or not os.path.isabs(cand)):
            return cand
    return "nvcc"


def stale():
    if not LIB.exists():
        return True
    t = LIB.stat().st_mtime
    return any(p.stat().st_mtime > t for p in DEPS)


def object_stale(obj, depfile):
    """Whether obj is older than a file its last compilation read."""
    if not obj.exists() or not depfile.exists():
        return True
    named = depfile.read_text().split(":", 1)[1].replace("\\\n", " ").split()
    t = obj.stat().st_mtime
    return any(not os.path.exists(p) or os.stat(p).st_mtime > t for p in named if not p.startswith("/usr/"))


def build(force=False, verbose=False):
    if not force and not stale():
        return LIB
    OBJ_DIR.mkdir(exist_ok=True)
    objects, running = [], []
    for src in SOURCES:
        obj, dep = OBJ_DIR / (src.stem + ".o"), OBJ_DIR / (src.stem + ".d")
        objects.append(str(obj))
        if not force and not object_stale(obj, dep):
            continue
        cmd = [nvcc(), *NVCC_FLAGS, "-MMD", "-MF", str(dep), "-c", "-o", str(obj), str(src)]
        if verbose:
            print(" ".join(cmd), flush=True)
        running.append((cmd, obj, subprocess.Popen(cmd)))
    failed = [(cmd, obj) for cmd, obj, p in running if p.wait() != 0]
    for cmd, obj in failed:
        obj.unlink(missing_ok=True)
    if failed:
        raise subprocess.CalledProcessError(1, failed[0][0])
    cmd = [nvcc(), *NVCC_FLAGS, "-shared", "-o", str(LIB) + ".tmp", *objects]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(str(LIB) + ".tmp", LIB)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
    print(LIB)
