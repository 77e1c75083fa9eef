"""Builds libhelion_lce.so (hand-written CUDA for sm_100a) in-tree with nvcc.

The library has a plain C ABI (include/helion_lce.h) and no dependency on torch headers, so it
builds in seconds and is loaded with ctypes. ``python -m helion_b200.build`` rebuilds it.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import tempfile
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
LIB_DIR = PKG_DIR / "_lib"
LIB_PATH = LIB_DIR / "libhelion_lce.so"
SOURCES = [CSRC / "lce_api.cu", CSRC / "linear_api.cu", CSRC / "block_api.cu"]
HEADERS = sorted(CSRC.glob("*.cuh")) + [PKG_DIR.parent / "include" / "helion_lce.h"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC",
]


def find_nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found; set NVCC or put it on PATH to build libhelion_lce.so")
    return cand


def is_stale() -> bool:
    if not LIB_PATH.exists():
        return True
    built = LIB_PATH.stat().st_mtime
    return any(p.stat().st_mtime > built for p in SOURCES + HEADERS)


def build_library(force: bool = False, verbose: bool = False) -> Path:
    """Compile the shared library if it is missing or older than its sources."""
    if not force and not is_stale():
        return LIB_PATH
    LIB_DIR.mkdir(exist_ok=True)
    flags = [*NVCC_FLAGS, *(["-Xptxas", "-v"] if verbose else [])]
    with tempfile.TemporaryDirectory(dir=LIB_DIR) as tmp:
        objects = [Path(tmp) / f"{src.stem}.o" for src in SOURCES]
        # one nvcc per source, side by side
        procs = [subprocess.Popen([find_nvcc(), *flags, "-c", "-o", str(obj), str(src)], stdout=subprocess.PIPE,
                                  stderr=subprocess.STDOUT, text=True) for src, obj in zip(SOURCES, objects)]
        outputs = [proc.communicate()[0] for proc in procs]
        for proc, out in zip(procs, outputs):
            if proc.returncode != 0:
                raise RuntimeError(f"nvcc failed ({proc.returncode}):\n{out}")
            if verbose:
                sys.stderr.write(out)
        # linked beside its place and renamed into it: a process that loads the library never sees half a file
        linked = Path(tmp) / LIB_PATH.name
        link = subprocess.run([find_nvcc(), "-shared", *NVCC_FLAGS, "-o", str(linked), *map(str, objects)],
                              capture_output=True, text=True)
        if link.returncode != 0:
            raise RuntimeError(f"nvcc failed ({link.returncode}):\n{link.stdout}\n{link.stderr}")
        linked.replace(LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    print(build_library(force=True, verbose="-v" in sys.argv))
