"""Build ``libpiper_merge.so`` and ``libpiper_fp4.so`` in-tree with nvcc for sm_100a, and the latter's calls with g++.

Usage: ``python -m piper_offload_b200.build`` (also called by
``__graft_entry__.build()``). A library newer than every source file of its
own is left as it is, the calls if they were also built for this interpreter
and torch.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
SOURCES = [PKG / "csrc" / "merge.cu"]
DEPS = SOURCES + [PKG / "csrc" / "ptx.cuh", PKG / "csrc" / "numerics.cuh", ROOT / "include" / "piper_merge.h"]
OUT = PKG / "libpiper_merge.so"
FP4_SOURCES = [PKG / "csrc" / "fp4.cu"]
FP4_DEPS = FP4_SOURCES + [
    *(PKG / "csrc" / n for n in ("fp4_quant.cuh", "fp4_tiles.cuh", "fp4_linear.cuh", "fp4_grad.cuh", "fp4_ptx.cuh", "ptx.cuh", "numerics.cuh")),
    ROOT / "include" / "piper_fp4.h",
]
FP4_OUT = PKG / "libpiper_fp4.so"
CALLS_SOURCES = [PKG / "csrc" / "fp4_calls.cpp"]
CALLS_DEPS = CALLS_SOURCES + [ROOT / "include" / "piper_fp4.h"]
CALLS_OUT = PKG / "_fp4_calls.so"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo",
    "-O3",
    "-std=c++17",
    "--fmad=false",  # only the explicit fmaf() calls fuse, matching the reference's rounding points
    "-Xcompiler", "-fPIC",
    "-shared",
    # No --split-compile: its parallel device optimisation gave a different
    # binary on every build of the same source (instantiations measured up to
    # 20 % apart on a B200); one thread gives the same code each time.
]


def nvcc() -> str:
    cand = os.environ.get("NVCC") or "/usr/local/cuda/bin/nvcc"
    return cand if Path(cand).exists() else shutil.which("nvcc") or "nvcc"


def up_to_date(out: Path = OUT, deps: list[Path] = DEPS) -> bool:
    if not out.exists():
        return False
    t = out.stat().st_mtime
    return all(p.stat().st_mtime <= t for p in deps)


def _compile(out: Path, sources: list[Path], verbose: bool) -> None:
    tmp = out.with_suffix(".so.tmp")
    cmd = [nvcc(), *NVCC_FLAGS, "-o", str(tmp), *map(str, sources)]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True, cwd=str(ROOT))
    os.replace(tmp, out)


def build(force: bool = False, verbose: bool = False) -> Path:
    """The merges' library, and then the FP4 operators' beside it."""
    if force or not up_to_date():
        _compile(OUT, SOURCES, verbose)
    build_fp4(force, verbose)
    return OUT


def build_fp4(force: bool = False, verbose: bool = False) -> Path:
    if force or not up_to_date(FP4_OUT, FP4_DEPS):
        _compile(FP4_OUT, FP4_SOURCES, verbose)
    build_calls(force, verbose)
    return FP4_OUT


def build_calls(force: bool = False, verbose: bool = False) -> Path:
    """The operators' calls from Python: host code against this interpreter's torch, which is noted beside it."""
    import torch

    fits = f"{sysconfig.get_config_var('SOABI')} torch {torch.__version__} abi {int(torch._C._GLIBCXX_USE_CXX11_ABI)}"
    note = CALLS_OUT.with_suffix(".so.fits")
    if force or not up_to_date(CALLS_OUT, CALLS_DEPS) or not note.exists() or note.read_text() != fits:
        base = Path(torch.__file__).resolve().parent
        tmp = CALLS_OUT.with_suffix(".so.tmp")
        cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
               f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
               *(f"-I{d}" for d in (base / "include", base / "include" / "torch" / "csrc" / "api" / "include",
                                    Path(nvcc()).resolve().parents[1] / "include", sysconfig.get_paths()["include"])),
               "-o", str(tmp), *map(str, CALLS_SOURCES), f"-L{base / 'lib'}", "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True, cwd=str(ROOT))
        os.replace(tmp, CALLS_OUT)
        note.write_text(fits)
    return CALLS_OUT


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(OUT)
    print(FP4_OUT)
    print(CALLS_OUT)
