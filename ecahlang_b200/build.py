"""Build the in-tree CUDA library ``lib/libecah_sampler.so`` for sm_100a.

The library is plain CUDA C++ behind an ``extern "C"`` ABI
(include/ecah_sampler.h); it links the CUDA runtime statically and has no
torch dependency, so any FFI (ctypes here) can load it.
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
LIB_DIR = os.path.join(PKG, "lib")
LIB = os.path.join(LIB_DIR, "libecah_sampler.so")
OBJ_DIR = os.path.join(LIB_DIR, "build")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
         "-Xcompiler", "-fvisibility=hidden", "--expt-relaxed-constexpr"]
SOURCES = ["sampler.cu", "noalloc.cu", "diag.cu", "logprobs.cu", "paged_append.cu", "paged_decode.cu"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; the sampler is CUDA-only and has no fallback")


def _stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = glob.glob(os.path.join(CSRC, "*")) + glob.glob(os.path.join(ROOT, "include", "*.h"))
    return any(os.path.getmtime(d) > t for d in deps)


def _object(source: str, force: bool, verbose: bool) -> str:
    """Compile one source, unless its object is newer than everything the last
    compilation read (nvcc's own dependency list)."""
    obj = os.path.join(OBJ_DIR, source + ".o")
    dep = obj + ".d"
    if not force and os.path.exists(obj) and os.path.exists(dep):
        read = [d for d in open(dep).read().replace("\\\n", " ").split(":", 1)[-1].split() if d.startswith(ROOT)]
        if read and all(os.path.exists(d) and os.path.getmtime(d) <= os.path.getmtime(obj) for d in read):
            return obj
    cmd = [_nvcc(), *ARCH, *FLAGS, "-I", os.path.join(ROOT, "include"), "-MD", "-MF", dep, "-c",
           "-o", obj, os.path.join(CSRC, source)]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
        print(" ".join(cmd))
    subprocess.run(cmd, check=True)
    return obj


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile the library if a source is newer than it; returns its path."""
    if not force and not _stale():
        return LIB
    os.makedirs(OBJ_DIR, exist_ok=True)
    with ThreadPoolExecutor(len(SOURCES)) as pool:
        objects = list(pool.map(lambda s: _object(s, force, verbose), SOURCES))
    tmp = LIB + ".tmp"
    subprocess.run([_nvcc(), *ARCH, "-shared", "-o", tmp, *objects], check=True)
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    import sys
    print(build(force="--changed" not in sys.argv, verbose=True))
