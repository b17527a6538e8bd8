"""Build libb200tx.so (the sm_100a kernels and their C ABI) and its binding in-tree.

The library is compiled from ``csrc/b200tx.cu`` (which includes the kernel
headers next to it) with nvcc for ``sm_100a`` only and written to
``solution/_lib/libb200tx.so``, where :mod:`solution._native` loads it.
``csrc/decode_binding.cpp``, the Python calls of the decoding operators, is
compiled with g++ against torch's headers and written next to it, where
:mod:`solution._binding` loads it.
Run ``python build_native.py`` or call :func:`build`.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PACKAGE_DIR = Path(__file__).resolve().parent
CSRC_DIR = PACKAGE_DIR / "csrc"
INCLUDE_DIR = PACKAGE_DIR.parent / "include"
LIB_DIR = PACKAGE_DIR / "solution" / "_lib"
LIB_PATH = LIB_DIR / "libb200tx.so"
BINDING_SOURCE = CSRC_DIR / "decode_binding.cpp"
BINDING_PATH = LIB_DIR / "_decode_binding.so"

NVCC_FLAGS = (
    "-gencode",
    "arch=compute_100a,code=sm_100a",
    "-O3",
    "-lineinfo",
    "-std=c++17",
    "-Xcompiler",
    "-fPIC",
    "-shared",
)


def _nvcc() -> str:
    candidates = [
        os.environ.get("NVCC"),
        shutil.which("nvcc"),
        "/usr/local/cuda/bin/nvcc",
    ]
    for candidate in candidates:
        if candidate and Path(candidate).exists():
            return candidate
    raise RuntimeError("nvcc not found; set NVCC or put the CUDA toolkit on PATH")


def _sources() -> list[Path]:
    return sorted(CSRC_DIR.glob("*.cu")) + sorted(CSRC_DIR.glob("*.cuh")) + [
        INCLUDE_DIR / "b200tx.h"
    ]


def _stale(target: Path, sources: list[Path]) -> bool:
    if not target.exists():
        return True
    built = target.stat().st_mtime
    return any(source.stat().st_mtime > built for source in sources)


def is_stale() -> bool:
    """Return whether the library is missing or older than any source file."""

    return _stale(LIB_PATH, _sources())


def binding_is_stale() -> bool:
    """Return whether the binding is missing or older than its sources."""

    return _stale(BINDING_PATH, [BINDING_SOURCE, INCLUDE_DIR / "b200tx.h"])


def _run(command: list[str], tmp: Path, target: Path, verbose: bool) -> None:
    if verbose:
        print(" ".join(command), flush=True)
    result = subprocess.run(command, capture_output=True, text=True)
    if result.returncode != 0:
        raise RuntimeError(
            f"{Path(command[0]).name} failed building {target.name}:\n" + result.stdout + result.stderr
        )
    os.replace(tmp, target)


def build_binding(force: bool = False, verbose: bool = False) -> Path:
    """Compile the binding if it is missing or stale; return its path."""

    if not force and not binding_is_stale():
        return BINDING_PATH
    import torch  # noqa: PLC0415 - only the build needs its headers here

    LIB_DIR.mkdir(parents=True, exist_ok=True)
    torch_dir = Path(torch.__file__).resolve().parent
    cuda = Path(_nvcc()).resolve().parents[1]
    includes = (
        INCLUDE_DIR,
        torch_dir / "include",
        torch_dir / "include" / "torch" / "csrc" / "api" / "include",
        Path(sysconfig.get_paths()["include"]),
        cuda / "include",
    )
    tmp = BINDING_PATH.with_suffix(".so.tmp")
    command = [
        shutil.which(os.environ.get("CXX", "g++")) or "g++",
        "-O2",
        "-std=c++17",
        "-fPIC",
        "-shared",
        "-fvisibility=hidden",
        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
        *(f"-I{path}" for path in includes),
        "-o",
        str(tmp),
        str(BINDING_SOURCE),
        f"-L{torch_dir / 'lib'}",
        "-ltorch_python",
        "-ltorch",
        "-ltorch_cpu",
        "-lc10",
        "-lc10_cuda",
    ]
    _run(command, tmp, BINDING_PATH, verbose)
    return BINDING_PATH


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile the library and its binding where missing or stale; return the library's path."""

    build_binding(force, verbose)
    if not force and not is_stale():
        return LIB_PATH
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    tmp = LIB_PATH.with_suffix(".so.tmp")
    command = [
        _nvcc(),
        *NVCC_FLAGS,
        f"-I{INCLUDE_DIR}",
        "-o",
        str(tmp),
        str(CSRC_DIR / "b200tx.cu"),
    ]
    _run(command, tmp, LIB_PATH, verbose)
    return LIB_PATH


if __name__ == "__main__":
    path = build(force="--force" in sys.argv, verbose=True)
    print(path)
