"""Build the sm_100a shared library ``llamamps_b200/lib/libllamamps_b200.so``.

Every ``csrc/*.cu`` file is compiled by nvcc for ``sm_100a`` only and linked
into one C-ABI shared library (declared in ``include/llamamps_b200.h``).  The
library is built in-tree so it ships with the source checkout; objects go to
``llamamps_b200/_build/``.  ``csrc/bind_q4.cpp`` becomes the Python extension
``llamamps_b200/lib/bind_q4.so`` (the 4-bit KV cache's eager calls), compiled
by the host compiler against the installed torch.

    python -m llamamps_b200.build [--force] [--verbose]
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import hashlib
import os
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
BUILD = os.path.join(PKG, "_build")
LIBDIR = os.path.join(PKG, "lib")
LIB_NAME = "libllamamps_b200.so"
LIB_PATH = os.path.join(LIBDIR, LIB_NAME)
BIND_PATH = os.path.join(LIBDIR, "bind_q4.so")

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH_FLAGS + [
    "-O3", "-lineinfo", "-std=c++17", "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC,-O3", "-I", INCLUDE,
]


def nvcc_path() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found: the CUDA toolkit is required to build llamamps_b200")
    return cand


def _sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _headers():
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    hs += [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE) if f.endswith(".h")]
    return sorted(hs)


def _digest(paths, extra=""):
    h = hashlib.sha256(extra.encode())
    for p in paths:
        with open(p, "rb") as f:
            h.update(p.encode())
            h.update(f.read())
    return h.hexdigest()


def _compile(nvcc, src, obj, verbose):
    cmd = [nvcc, *NVCC_FLAGS, "-c", src, "-o", obj]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed on {os.path.basename(src)}:\n{r.stdout}\n{r.stderr}")
    return r.stderr if verbose else ""


def build_binding(force: bool = False) -> str:
    """Compile the Python extension of csrc/bind_q4.cpp (if it, the header or torch changed)."""
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths
    src = os.path.join(CSRC, "bind_q4.cpp")
    flags = ["-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
             f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
             f'-DLMPS_TORCH_VERSION="{torch.__version__}"']
    stamp = os.path.join(LIBDIR, ".bind_stamp")
    digest = _digest([src, os.path.join(INCLUDE, "llamamps_b200.h")],
                     " ".join(flags) + torch.__version__ + sys.version)
    if not force and os.path.exists(BIND_PATH) and os.path.exists(stamp):
        with open(stamp) as f:
            if f.read().strip() == digest:
                return BIND_PATH
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc_path())))
    inc = [*include_paths(), sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    tmp = BIND_PATH + ".tmp"
    os.makedirs(LIBDIR, exist_ok=True)
    r = subprocess.run([shutil.which("g++") or "g++", *flags, *[f"-I{i}" for i in inc], src, "-o", tmp, f"-L{libs}",
                        "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"], capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on bind_q4.cpp:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, BIND_PATH)
    with open(stamp, "w") as f:
        f.write(digest)
    return BIND_PATH


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile (if sources changed) and return the library path."""
    with cf.ThreadPoolExecutor(max_workers=1) as ex:
        binding = ex.submit(build_binding, force)
        path = _build_library(force, verbose)
        binding.result()
    return path


def _build_library(force: bool, verbose: bool) -> str:
    srcs = _sources()
    stamp = os.path.join(LIBDIR, ".build_stamp")
    digest = _digest(srcs + _headers(), " ".join(NVCC_FLAGS))
    if not force and os.path.exists(LIB_PATH) and os.path.exists(stamp):
        with open(stamp) as f:
            if f.read().strip() == digest:
                return LIB_PATH
    os.makedirs(BUILD, exist_ok=True)
    os.makedirs(LIBDIR, exist_ok=True)
    nvcc = nvcc_path()
    objs = [os.path.join(BUILD, os.path.basename(s)[:-3] + ".o") for s in srcs]
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        futs = [ex.submit(_compile, nvcc, s, o, verbose) for s, o in zip(srcs, objs)]
        for fut in futs:
            out = fut.result()
            if out:
                sys.stderr.write(out)
    tmp = LIB_PATH + ".tmp"
    r = subprocess.run([nvcc, *ARCH_FLAGS, "-shared", "-o", tmp, *objs, "-lcuda"],
                       capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB_PATH)
    with open(stamp, "w") as f:
        f.write(digest)
    return LIB_PATH


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose))
