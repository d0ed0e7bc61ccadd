"""Build ``libpiper_merge.so`` and ``libpiper_fp4.so`` in-tree with nvcc for sm_100a.

Usage: ``python -m piper_offload_b200.build`` (also called by
``__graft_entry__.build()``). A library newer than every source file of its
own is left as it is.
"""

from __future__ import annotations

import os
import subprocess
import sys
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
    return cand if Path(cand).exists() else "nvcc"


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
    """The merges' library; the FP4 operators' is built beside it."""
    build_fp4(force, verbose)
    if force or not up_to_date():
        _compile(OUT, SOURCES, verbose)
    return OUT


def build_fp4(force: bool = False, verbose: bool = False) -> Path:
    if force or not up_to_date(FP4_OUT, FP4_DEPS):
        _compile(FP4_OUT, FP4_SOURCES, verbose)
    return FP4_OUT


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(OUT)
    print(FP4_OUT)
