"""ctypes binding of ``libpiper_fp4.so`` (the sm_100a C ABI in ``include/piper_fp4.h``).

As with the merges there is no fallback: a missing library raises
``RuntimeError`` at the first call.
"""

from __future__ import annotations

import ctypes
import os
import threading
from pathlib import Path
from typing import Any

import torch

from ._native import ETIMEOUT, EINVAL, OK, current_stream_handle

LIB_PATH = Path(__file__).resolve().parent / "libpiper_fp4.so"

FMT_MX = 0
FMT_NV = 1
DT_BF16 = 0
DT_F32 = 2
SECOND_NONE = 0
SECOND_GIVEN = 1
SECOND_COMPUTE = 2
SMALL_MATRIX = 65536  # PIPER_FP4_SMALL_MATRIX

EXPORTED_SYMBOLS = (
    "piper_fp4_quantize",
    "piper_fp4_dequantize",
    "piper_fp4_linear_workspace",
    "piper_fp4_grad_input_workspace",
    "piper_fp4_linear",
    "piper_fp4_grad_input",
    "piper_fp4_linear_plan",
    "piper_fp4_grad_input_plan",
    "piper_fp4_last_error",
    "piper_fp4_device_status",
    "piper_fp4_version",
    "piper_fp4_launches",
)


class Matrix(ctypes.Structure):
    """Mirror of ``piper_fp4_matrix``."""

    _fields_ = [
        ("codes", ctypes.c_void_p),
        ("scale", ctypes.c_void_p),
        ("second", ctypes.c_void_p),
        ("batch", ctypes.c_int64),
        ("rows", ctypes.c_int64),
        ("cols", ctypes.c_int64),
        ("format", ctypes.c_int32),
        ("swizzled", ctypes.c_int32),
    ]


class Plan(ctypes.Structure):
    """Mirror of ``piper_fp4_plan``."""

    _fields_ = [("tile_tokens", ctypes.c_int32), ("tile_columns", ctypes.c_int32), ("split", ctypes.c_int32),
                ("fused", ctypes.c_int32)]


_lib = None
_lock = threading.Lock()


def library_path() -> Path:
    return Path(os.environ.get("PIPER_FP4_LIB", LIB_PATH))


def load() -> ctypes.CDLL:
    """Load the native library (once) and declare its signatures."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        path = library_path()
        if not path.exists():
            raise RuntimeError(
                f"native FP4 library {path} is missing; build it with "
                "`python -c 'import __graft_entry__ as g; g.build()'` (there is no CPU fallback)."
            )
        lib = ctypes.CDLL(str(path))
        vp, i32, i64, sz = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_size_t
        mat = ctypes.POINTER(Matrix)
        lib.piper_fp4_quantize.argtypes = [mat, vp, i64, i32, i32, i32, vp, vp]
        lib.piper_fp4_dequantize.argtypes = [mat, vp, i32, vp]
        lib.piper_fp4_linear_workspace.argtypes = [mat, i64, ctypes.POINTER(sz)]
        lib.piper_fp4_grad_input_workspace.argtypes = [mat, vp, i64, i64, i32, ctypes.POINTER(sz)]
        lib.piper_fp4_linear.argtypes = [mat, vp, i64, i64, vp, vp, i32, vp, i32, vp, sz, vp]
        lib.piper_fp4_grad_input.argtypes = [mat, vp, i64, i64, vp, vp, i32, vp, sz, vp]
        lib.piper_fp4_linear_plan.argtypes = [mat, i64, ctypes.POINTER(Plan)]
        lib.piper_fp4_grad_input_plan.argtypes = [mat, i64, i32, i32, ctypes.POINTER(Plan)]
        lib.piper_fp4_device_status.argtypes = [vp, ctypes.POINTER(ctypes.c_uint32)]
        for name in EXPORTED_SYMBOLS[:8] + ("piper_fp4_device_status",):
            getattr(lib, name).restype = ctypes.c_int
        lib.piper_fp4_last_error.restype = ctypes.c_char_p
        lib.piper_fp4_version.restype = ctypes.c_char_p
        lib.piper_fp4_launches.restype = ctypes.c_uint64
        _lib = lib
        return lib


_calls = None


def calls() -> Any:
    """The compiled calls (``csrc/fp4_calls.cpp``), bound to the library's entry points. Loads both once."""
    global _calls
    if _calls is None:
        lib = load()
        try:
            from . import _fp4_calls as module
        except ImportError as exc:
            raise RuntimeError("the FP4 operators' compiled calls are missing or do not fit this torch; build them with "
                               "`python -c 'import __graft_entry__ as g; g.build()'`.") from exc
        module.bind(getattr(torch, "float4_e2m1fn_x2", None),
                    *(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in EXPORTED_SYMBOLS[:6]))
        _calls = module
    return _calls


def check(rc: int) -> None:
    if rc == OK:
        return
    msg = load().piper_fp4_last_error().decode("utf-8", "replace")
    if rc == EINVAL:
        raise ValueError(msg)
    raise RuntimeError(f"piper fp4 failed (status {rc}): {msg}")


# The current stream's handle by device index, without making a stream object (2 us of a 10 us call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def raw_stream(index: int) -> int:
    return _raw_stream(index) if _raw_stream is not None else current_stream_handle(torch.device("cuda", index))


def device_status(device: torch.device) -> int:
    """Read and clear the device-side status word (synchronises the current stream)."""
    out = ctypes.c_uint32(0)
    with torch.cuda.device(device):
        rc = load().piper_fp4_device_status(current_stream_handle(device), ctypes.byref(out))
    if rc not in (OK, ETIMEOUT):
        check(rc)
    return int(out.value)


def version() -> str:
    return load().piper_fp4_version().decode()


def linear_plan(m: Matrix, tokens: int) -> Plan:
    """How the product of a matrix (or a stack of them) and ``tokens`` tokens runs on the current device."""
    plan = Plan()
    check(load().piper_fp4_linear_plan(ctypes.byref(m), tokens, ctypes.byref(plan)))
    return plan


def grad_input_plan(m: Matrix, tokens: int, *, grouped: bool, dtype: int) -> Plan:
    """How the product's gradient runs."""
    plan = Plan()
    check(load().piper_fp4_grad_input_plan(ctypes.byref(m), tokens, grouped, dtype, ctypes.byref(plan)))
    return plan


def launches() -> int:
    """Kernels launched by this process through the library so far."""
    return int(load().piper_fp4_launches())
