"""Build the C-ABI library `libvdexec.so` for sm_100a with nvcc (in-tree).

    python -m verdict_b200.build [--verbose]

The library links the CUDA runtime statically and reaches the driver API
(tensor-map encoding) through cudaGetDriverEntryPoint, so it needs no torch and
no libcuda at link time.
"""

from __future__ import annotations

import concurrent.futures
import hashlib
import importlib.util
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
# The torch binding of verdict_b200/ops.py, built beside the library where torch is installed.
TORCH_SOURCE = os.path.join(CSRC, "torch_ops.cpp")
TORCH_LIB = os.path.join(PKG, "_torch_ops.so")
# What each was built from.
HEADERS = [os.path.join(INCLUDE, "vdexec.h"), os.path.join(INCLUDE, "vdexec_kernels.h")]
LIB_STAMP = os.path.join(OBJ, "libvdexec.stamp")
TORCH_STAMP = os.path.join(OBJ, "torch_ops.stamp")

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
    return all(os.path.getmtime(p) <= t for p in DEPS if os.path.exists(p) and p != TORCH_SOURCE)


def _digest(paths, *more: str) -> str:
    h = hashlib.sha256()
    for p in paths:
        with open(p, "rb") as f:
            h.update(hashlib.sha256(f.read()).digest())
    for m in more:
        h.update(m.encode() + b"\0")
    return h.hexdigest()


def _read(path: str) -> str:
    try:
        with open(path) as f:
            return f.read().strip()
    except OSError:
        return ""


def _write(path: str, text: str) -> None:
    with open(path, "w") as f:
        f.write(text + "\n")


def library_has_this_header() -> bool:
    """Whether libvdexec.so was built with the C entries as include/ declares them now."""
    return up_to_date() or _read(LIB_STAMP) == _digest(HEADERS)


def _torch_digest() -> str:
    """What the torch binding depends on: its source, the C entries it calls, and the torch and Python it is built for."""
    import torch

    return _digest([TORCH_SOURCE, *HEADERS], torch.__version__, str(torch.version.cuda), sys.implementation.cache_tag)


def torch_up_to_date() -> bool:
    return os.path.exists(TORCH_LIB) and _read(TORCH_STAMP) == _torch_digest()


def build_torch_ops(force: bool = False, verbose: bool = False) -> str:
    """Compile verdict_b200/_torch_ops.so against the installed torch; it links libvdexec.so beside it."""
    if not force and torch_up_to_date():
        return TORCH_LIB
    import sysconfig

    from torch.utils import cpp_extension
    import torch

    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", "-I", INCLUDE,
           "-I", sysconfig.get_paths()["include"], "-I", os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include")]
    for path in cpp_extension.include_paths():
        cmd += ["-isystem", path]
    for path in cpp_extension.library_paths():
        cmd += ["-L", path]
    cmd += [TORCH_SOURCE, "-o", TORCH_LIB + ".tmp", "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_python",
            "-L", PKG, "-l:libvdexec.so", "-Wl,-rpath,$ORIGIN"]
    digest = _torch_digest()
    _run(cmd, verbose)
    os.makedirs(OBJ, exist_ok=True)
    _write(TORCH_STAMP, "")  # until the new file is in place
    os.replace(TORCH_LIB + ".tmp", TORCH_LIB)
    _write(TORCH_STAMP, digest)
    return TORCH_LIB


def _run(cmd: list, verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
    if verbose:
        print(res.stdout + res.stderr)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date():
        return LIB
    os.makedirs(OBJ, exist_ok=True)
    digest = _digest(HEADERS)
    objects = [os.path.join(OBJ, os.path.splitext(os.path.basename(src))[0] + ".o") for src in SOURCES]
    flags = [*NVCC_FLAGS, *(["-Xptxas=-v"] if verbose else []), "-I", INCLUDE, "-I", CSRC]
    with concurrent.futures.ThreadPoolExecutor(len(SOURCES)) as pool:
        list(pool.map(lambda so: _run([nvcc(), *flags, "-c", so[0], "-o", so[1]], verbose), zip(SOURCES, objects)))
    _run([nvcc(), *NVCC_FLAGS, "-shared", *objects, "-o", LIB + ".tmp"], verbose)
    _write(LIB_STAMP, "")
    os.replace(LIB + ".tmp", LIB)
    _write(LIB_STAMP, digest)
    return LIB


if __name__ == "__main__":
    print(build(force=True, verbose="--verbose" in sys.argv))
    if importlib.util.find_spec("torch") is not None:
        print(build_torch_ops(force=True, verbose="--verbose" in sys.argv))
