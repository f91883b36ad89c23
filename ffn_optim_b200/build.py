"""Builds the in-tree CUDA library ``ffn_optim_b200/_lib/libffn_b200.so`` for sm_100a.

The library is the C-ABI declared in ``include/ffn_b200.h``; the Python host layer loads it
with ctypes.  It is built with nvcc directly (no torch extension machinery), so the result
is a plain shared object that any host language can bind.
"""
from __future__ import annotations

import hashlib
import os
import re
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIBDIR = PKG / "_lib"
LIB = LIBDIR / "libffn_b200.so"
SOURCES = [CSRC / "ffn_capi.cu", CSRC / "ffn_noalloc.cu", CSRC / "ffn_placement.cu", CSRC / "ffn_quant.cu",
           CSRC / "ffn_layers.cu"]
HEADERS = [CSRC / "ffn_kernel.cuh", CSRC / "ffn_rowblock.cuh", CSRC / "ffn_hslice.cuh", CSRC / "gemm_kernel.cuh",
           CSRC / "pack_kernel.cuh",
           CSRC / "stream_kernel.cuh", CSRC / "router_kernel.cuh", ROOT / "include" / "ffn_b200.h"]
ARCH = "-gencode=arch=compute_100a,code=sm_100a"
# -fvisibility=hidden keeps the template kernels private; the extern "C" API is exported
# through the FFN_B200_EXPORT default-visibility attribute in the header.
FLAGS = [ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: the ffn_b200 CUDA library cannot be built")


def source_digest() -> str:
    h = hashlib.sha256(" ".join(FLAGS).encode())
    for path in SOURCES + HEADERS:
        h.update(path.read_bytes())
    return h.hexdigest()


def stamp_path() -> Path:
    return LIBDIR / "libffn_b200.sha256"


def up_to_date() -> bool:
    return LIB.exists() and stamp_path().exists() and stamp_path().read_text().strip() == source_digest()


def _included(path: Path, seen: set) -> set:
    """``path`` and the in-tree files it includes, transitively."""
    if path not in seen:
        seen.add(path)
        for name in re.findall(r'^#include "([^"]+)"', path.read_text(), re.M):
            _included((path.parent / name).resolve(), seen)
    return seen


def _compile(source: Path, force: bool, verbose: bool) -> Path:
    """The object file of one source, compiled if it, a file it includes, the flags or the compiler changed."""
    obj = LIBDIR / (source.stem + ".o")
    stamp = LIBDIR / (source.stem + ".o.sha256")
    version = subprocess.run([nvcc(), "--version"], capture_output=True, text=True).stdout
    h = hashlib.sha256(" ".join(FLAGS + [version]).encode())
    for path in sorted(_included(source.resolve(), set())):
        h.update(path.read_bytes())
    digest = h.hexdigest()
    if not force and obj.exists() and stamp.exists() and stamp.read_text().strip() == digest:
        return obj
    tmp = obj.with_suffix(f".{os.getpid()}.tmp")  # (an interrupted compilation must not pass for the object)
    cmd = [nvcc(), *FLAGS, "-c", "-Xptxas", "-v" if verbose else "-O3", "-I", str(ROOT / "include"), "-o", str(tmp),
           str(source)]
    try:
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError("nvcc failed:\n" + " ".join(cmd) + "\n" + res.stdout + res.stderr)
        stamp.unlink(missing_ok=True)  # never beside an object of other sources
        tmp.replace(obj)
    finally:
        tmp.unlink(missing_ok=True)
    if verbose:
        sys.stderr.write(res.stdout + res.stderr)
    stamp.write_text(digest + "\n")
    return obj


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile the library if its sources changed; returns the library path."""
    if not force and up_to_date():
        return LIB
    LIBDIR.mkdir(exist_ok=True)
    with ThreadPoolExecutor(len(SOURCES)) as pool:
        objects = list(pool.map(lambda src: _compile(src, force, verbose), SOURCES))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [nvcc(), ARCH, "--shared", "-o", str(tmp)] + [str(o) for o in objects]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + " ".join(cmd) + "\n" + res.stdout + res.stderr)
    stamp_path().unlink(missing_ok=True)
    tmp.replace(LIB)
    stamp_path().write_text(source_digest() + "\n")
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
