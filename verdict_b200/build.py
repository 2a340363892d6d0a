"""Build the C-ABI library `libvdexec.so` for sm_100a with nvcc (in-tree).

    python -m verdict_b200.build [--verbose]

The library links the CUDA runtime statically and reaches the driver API
(tensor-map encoding) through cudaGetDriverEntryPoint, so it needs no torch and
no libcuda at link time.
"""

from __future__ import annotations

import concurrent.futures
import os
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(REPO, "include")
LIB = os.path.join(PKG, "libvdexec.so")
SOURCES = [os.path.join(CSRC, "vdexec.cu"), os.path.join(CSRC, "operators.cu")]
DEPS = ([os.path.join(CSRC, f) for f in os.listdir(CSRC)]
        + [os.path.join(INCLUDE, "vdexec.h"), os.path.join(INCLUDE, "vdexec_kernels.h")])
OBJ = os.path.join(PKG, "_build")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC,-O3,-fvisibility=hidden",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def up_to_date() -> bool:
    if not os.path.exists(LIB):
        return False
    t = os.path.getmtime(LIB)
    return all(os.path.getmtime(p) <= t for p in DEPS if os.path.exists(p))


def _run(cmd: list, verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
    if verbose:
        print(res.stdout + res.stderr)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date():
        return LIB
    os.makedirs(OBJ, exist_ok=True)
    objects = [os.path.join(OBJ, os.path.splitext(os.path.basename(src))[0] + ".o") for src in SOURCES]
    flags = [*NVCC_FLAGS, *(["-Xptxas=-v"] if verbose else []), "-I", INCLUDE, "-I", CSRC]
    with concurrent.futures.ThreadPoolExecutor(len(SOURCES)) as pool:
        list(pool.map(lambda so: _run([nvcc(), *flags, "-c", so[0], "-o", so[1]], verbose), zip(SOURCES, objects)))
    _run([nvcc(), *NVCC_FLAGS, "-shared", *objects, "-o", LIB + ".tmp"], verbose)
    os.replace(LIB + ".tmp", LIB)
    return LIB


if __name__ == "__main__":
    print(build(force=True, verbose="--verbose" in sys.argv))
