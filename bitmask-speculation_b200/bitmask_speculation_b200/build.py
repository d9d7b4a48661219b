"""Build the sm_100a shared library in-tree with nvcc.

The library (``_lib/libbms_b200.so``) exports the C ABI of ``include/bms_b200.h``;
it is compiled ahead of time for ``sm_100a`` only (no JIT, no other targets) and
links the CUDA runtime statically, so it depends on the driver alone.
"""

from __future__ import annotations

import os
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent
SOURCE_ROOT = PACKAGE.parent / "csrc"
INCLUDE = PACKAGE.parents[1] / "include"
LIBRARY = PACKAGE / "_lib" / "libbms_b200.so"

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
              "-Xcompiler", "-fvisibility=hidden", "--expt-relaxed-constexpr"]
LINK_FLAGS = ["-shared", "-Xcompiler", "-fPIC"]


def sources() -> list[Path]:
    return sorted(p for p in SOURCE_ROOT.iterdir() if p.suffix in {".cu", ".cuh", ".h"}) + [
        INCLUDE / "bms_b200.h"]


def nvcc() -> str:
    cuda_home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    candidate = Path(cuda_home) / "bin" / "nvcc"
    if candidate.exists():
        return str(candidate)
    found = shutil.which("nvcc")
    if not found:
        raise RuntimeError("nvcc not found: the CUDA toolkit is required to build the library")
    return found


def stale() -> bool:
    if not LIBRARY.exists():
        return True
    built = LIBRARY.stat().st_mtime
    return any(p.stat().st_mtime > built for p in sources())


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile every ``csrc/*.cu`` (one nvcc each, side by side) into ``_lib/libbms_b200.so`` if stale."""
    if not force and not stale():
        return LIBRARY
    LIBRARY.parent.mkdir(parents=True, exist_ok=True)
    tmp = LIBRARY.with_suffix(f".{os.getpid()}.tmp")
    units = [p for p in sources() if p.suffix == ".cu"]
    objects = [LIBRARY.parent / f"{p.stem}.{os.getpid()}.o" for p in units]

    def compile_one(pair):
        flags = [*(["-Xptxas=-v"] if verbose else []), *ARCH_FLAGS, *NVCC_FLAGS]
        subprocess.run([nvcc(), *flags, "-I", str(INCLUDE), "-c", "-o", str(pair[1]), str(pair[0])], check=True)

    try:
        with ThreadPoolExecutor(len(units)) as pool:
            list(pool.map(compile_one, zip(units, objects)))
        subprocess.run([nvcc(), *ARCH_FLAGS, *LINK_FLAGS, "-o", str(tmp), *map(str, objects)], check=True)
        os.replace(tmp, LIBRARY)
    finally:
        for o in objects:
            o.unlink(missing_ok=True)
    return LIBRARY


if __name__ == "__main__":
    print(build(force=True, verbose=True))
