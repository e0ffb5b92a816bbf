"""Build the sampler's CUDA library in-tree (``b200_sampler/libns_sampler.so``).

    python -m b200_sampler.build          (from nano-inference_b200/)

nvcc cross-compiles for sm_100a only; no GPU is needed to build.  The library
is a plain shared object with a C ABI (``include/ns_sampler.h``,
``include/ns_losses.h``); it links the CUDA runtime statically and uses no
torch headers.  Every source has its own object under ``build/``: a change
to one compiles that one alone, a change to a header or to this file all of them.
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG_DIR)                     # nano-inference_b200/
REPO = os.path.dirname(ROOT)
CSRC = os.path.join(ROOT, "csrc")
INCLUDE = os.path.join(REPO, "include")
LIB_NAME = "libns_sampler.so"
LIB_PATH = os.path.join(PKG_DIR, LIB_NAME)

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC,-O2",
]
OBJ_DIR = os.path.join(ROOT, "build")


def nvcc_path() -> str:
    p = shutil.which("nvcc")
    if p:
        return p
    cand = "/usr/local/cuda/bin/nvcc"
    if os.path.exists(cand):
        return cand
    raise RuntimeError("nvcc not found")


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


HISTPACK_SRC = os.path.join(CSRC, "histpack.c")


def histpack_path() -> str:
    import sysconfig
    return os.path.join(PKG_DIR, "_histpack" + sysconfig.get_config_var("EXT_SUFFIX"))


def build_histpack(force: bool = False) -> str:
    """Compile the host-side history packer (a CPython extension, plain C)."""
    import sysconfig
    out = histpack_path()
    if not force and os.path.exists(out) and os.path.getmtime(out) >= os.path.getmtime(HISTPACK_SRC):
        return out
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        raise RuntimeError("no C compiler for the history packer")
    tmp = out + ".tmp"
    cmd = [cc, "-O3", "-shared", "-fPIC", "-I", sysconfig.get_paths()["include"], "-o", tmp, HISTPACK_SRC]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("gcc failed:\n" + r.stdout + r.stderr)
    os.replace(tmp, out)
    return out


def _headers():
    return glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h"))


def _common():
    """What every object depends on beside its source: all headers, since one
    may name another, and the flags, which stand in this file."""
    return [*_headers(), __file__]


def _deps():
    return sources() + _common()


def needs_build() -> bool:
    if not os.path.exists(LIB_PATH):
        return True
    t = os.path.getmtime(LIB_PATH)
    return any(os.path.getmtime(p) > t for p in _deps())


def _run(cmd, verbose: bool = False) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + r.stdout + r.stderr)
    if verbose:
        print(r.stdout + r.stderr)


def _compile(src: str, force: bool, verbose: bool) -> str:
    obj = os.path.join(OBJ_DIR, os.path.basename(src) + ".o")
    if not force and os.path.exists(obj) and all(os.path.getmtime(obj) >= os.path.getmtime(p)
                                                 for p in [src, *_common()]):
        return obj
    cmd = [nvcc_path(), *NVCC_FLAGS, "-I", INCLUDE, "-I", CSRC, "-c", "-o", obj + ".tmp", src]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    _run(cmd, verbose)
    os.replace(obj + ".tmp", obj)
    return obj


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile csrc/*.cu into the in-tree shared library (and the history
    packer); returns the library's path."""
    build_histpack(force)
    if not force and not needs_build():
        return LIB_PATH
    os.makedirs(OBJ_DIR, exist_ok=True)
    with ThreadPoolExecutor() as pool:
        objs = list(pool.map(lambda src: _compile(src, force, verbose), sources()))
    tmp = LIB_PATH + ".tmp"
    _run([nvcc_path(), *NVCC_FLAGS, "-shared", "-o", tmp, *objs], verbose)
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
