"""Build the native backend in-tree: ``metellus_b200/_lib/libmetellus_cuda.so``.

Run as ``python -m metellus_b200.csrc.build``. Uses nvcc for sm_100a; the library
links the CUDA runtime statically and NVRTC dynamically (rpath to the CUDA toolkit),
and resolves driver entry points at run time so it also loads on a machine without
a GPU driver (the CPU test suite checks its exported symbols there).
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent.parent
REPO = PKG.parent
LIB_DIR = PKG / "_lib"
LIB = LIB_DIR / "libmetellus_cuda.so"
PAGED = LIB_DIR / "_metellus_paged.so"   # the Python binding of the paged cache's operators
CUDA_HOME = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda"))
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    exe = shutil.which("nvcc") or str(CUDA_HOME / "bin" / "nvcc")
    if not Path(exe).exists():
        raise RuntimeError("nvcc not found; set CUDA_HOME")
    return exe


def sources() -> list[Path]:
    return sorted((PKG / "csrc").glob("*.cu"))


def build_backend(force: bool = False, verbose: bool = False) -> Path:
    """Compile every ``csrc/*.cu`` (in parallel, only what changed) and link them."""
    headers = [REPO / "include" / "metellus_b200.h", *(PKG / "csrc").glob("*.h"), *(PKG / "csrc").glob("*.cuh"),
               *(PKG / "csrc" / "include").glob("*.cuh")]
    newest_header = max(h.stat().st_mtime for h in headers)
    LIB_DIR.mkdir(exist_ok=True)
    newest = max(newest_header, *(s.stat().st_mtime for s in sources()))
    if not force and LIB.exists() and LIB.stat().st_mtime >= newest:
        build_binding(force, verbose)
        return LIB
    obj_dir = PKG / "csrc" / "_build"
    obj_dir.mkdir(exist_ok=True)

    def compile_one(src: Path) -> Path:
        obj = obj_dir / (src.stem + ".o")
        if not force and obj.exists() and obj.stat().st_mtime >= max(newest_header, src.stat().st_mtime):
            return obj
        cmd = [nvcc(), *ARCH_FLAGS, "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC", "-c",
               "-I", str(REPO / "include"), "-o", str(obj), str(src)]
        if verbose:
            print(" ".join(cmd))
        subprocess.run(cmd, check=True)
        return obj

    with ThreadPoolExecutor(max_workers=os.cpu_count() or 1) as pool:
        objects = list(pool.map(compile_one, sources()))
    cmd = [
        nvcc(), *ARCH_FLAGS, "-shared", "-Xcompiler", "-fPIC", "-o", str(LIB), *map(str, objects),
        "-cudart", "static", "-L", str(CUDA_HOME / "lib64"), "-lnvrtc",
        f"-Xlinker=-rpath,{CUDA_HOME / 'lib64'}",
    ]
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True)
    build_binding(force, verbose)
    return LIB


def build_binding(force: bool = False, verbose: bool = False) -> Path:
    """The CPython extension over the library's paged-cache entry points."""
    src, header = PKG / "csrc" / "python_paged.cpp", REPO / "include" / "metellus_b200.h"
    if not force and PAGED.exists() and PAGED.stat().st_mtime >= max(src.stat().st_mtime, header.stat().st_mtime):
        return PAGED
    cmd = [nvcc(), "-O3", "-std=c++17", "-shared", "-Xcompiler", "-fPIC", "-I", str(REPO / "include"),
           "-I", sysconfig.get_paths()["include"], "-o", str(PAGED), str(src), "-cudart", "none",
           "-L", str(LIB_DIR), "-lmetellus_cuda", "-Xlinker=-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True)
    return PAGED


if __name__ == "__main__":
    build_backend(force="--force" in sys.argv, verbose=True)
    print(LIB)
