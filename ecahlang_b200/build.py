"""Build the in-tree CUDA library ``lib/libecah_sampler.so`` for sm_100a.

The library is plain CUDA C++ behind an ``extern "C"`` ABI
(include/ecah_sampler.h); it links the CUDA runtime statically and has no
torch dependency, so any FFI (ctypes here) can load it.  ``lib/_ecah_binding.*.so``
is the torch side of the newer entry points: a CPython module that checks
tensors and calls the library; it is left out where there is no torch with CUDA.
"""
from __future__ import annotations

import glob
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sysconfig
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
LIB_DIR = os.path.join(PKG, "lib")
LIB = os.path.join(LIB_DIR, "libecah_sampler.so")


def binding_path() -> str:
    """The torch binding's file.  It depends on the ABIs of the interpreter and
    of torch, so it carries both names, and one built for others is not taken."""
    try:
        torch = importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:
        torch = "unknown"
    return os.path.join(LIB_DIR, f"_ecah_binding.{sysconfig.get_config_var('SOABI')}.torch-{torch}.so")


BINDING = binding_path()
OBJ_DIR = os.path.join(LIB_DIR, "build")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
         "-Xcompiler", "-fvisibility=hidden", "--expt-relaxed-constexpr"]
SOURCES = ["sampler.cu", "noalloc.cu", "diag.cu", "logprobs.cu", "paged_append.cu", "paged_decode.cu",
           "paged_prefill.cu", "paged_copy.cu", "drafts.cu"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; the sampler is CUDA-only and has no fallback")


def _stale(product: str) -> bool:
    if not os.path.exists(product):
        return True
    t = os.path.getmtime(product)
    deps = glob.glob(os.path.join(CSRC, "*")) + glob.glob(os.path.join(ROOT, "include", "*.h"))
    binding = os.path.join(CSRC, "binding.cpp")
    deps = [d for d in deps if (d == binding) == (product == BINDING) or d.endswith("ecah_sampler.h")]
    return any(os.path.getmtime(d) > t for d in deps)


def _torch():
    """Directory of a torch with CUDA (headers and libraries, without importing
    it), or None: the library needs none, its torch binding does."""
    spec = importlib.util.find_spec("torch")
    where = os.path.dirname(spec.origin) if spec and spec.origin else None
    return where if where and os.path.exists(os.path.join(where, "lib", "libtorch_cuda.so")) else None


def _build_binding(torch: str) -> None:
    cuda = os.path.dirname(os.path.dirname(_nvcc()))
    include = [os.path.join(ROOT, "include"), os.path.join(torch, "include"),
               os.path.join(torch, "include", "torch", "csrc", "api", "include"),
               sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
    tmp = BINDING + ".tmp"
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O2", "-fPIC", "-shared", "-fvisibility=hidden",
                    *(f"-I{d}" for d in include), os.path.join(CSRC, "binding.cpp"), "-o", tmp,
                    "-L" + os.path.join(torch, "lib"), "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda",
                    "-lc10", "-lc10_cuda"], check=True)
    os.replace(tmp, BINDING)


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
    """Compile the library and, beside a torch with CUDA, its torch binding, where a source is newer; returns the
    library's path."""
    torch = _torch()
    lib, binding = force or _stale(LIB), torch is not None and (force or _stale(BINDING))
    if not lib and not binding:
        return LIB
    os.makedirs(OBJ_DIR, exist_ok=True)
    with ThreadPoolExecutor(len(SOURCES) + 1) as pool:
        bound = pool.submit(_build_binding, torch) if binding else None
        if lib:
            objects = list(pool.map(lambda s: _object(s, force, verbose), SOURCES))
            tmp = LIB + ".tmp"
            subprocess.run([_nvcc(), *ARCH, "-shared", "-o", tmp, *objects], check=True)
            os.replace(tmp, LIB)
        if bound:
            bound.result()
    return LIB


if __name__ == "__main__":
    import sys
    changed = "--changed" in sys.argv        # only what a source is newer than
    print(build(force=not changed, verbose=True))
