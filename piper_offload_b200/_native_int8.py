"""ctypes binding of ``libpiper_int8.so`` (the sm_100a C ABI in ``include/piper_int8.h``).

As with the merges there is no fallback: a missing library raises
``RuntimeError`` at the first call.
"""

from __future__ import annotations

import ctypes
import os
import threading
from pathlib import Path

import torch

from ._native import ETIMEOUT, EINVAL, OK, current_stream_handle

LIB_PATH = Path(__file__).resolve().parent / "libpiper_int8.so"

DT_BF16 = 0
DT_F16 = 1
DT_F32 = 2
MAX_COLS = 65536  # PIPER_INT8_MAX_COLS

EXPORTED_SYMBOLS = (
    "piper_int8_linear_workspace",
    "piper_int8_grad_input_workspace",
    "piper_int8_linear",
    "piper_int8_grad_input",
    "piper_int8_linear_plan",
    "piper_int8_grad_input_plan",
    "piper_int8_last_error",
    "piper_int8_device_status",
    "piper_int8_version",
    "piper_int8_launches",
)


class Matrix(ctypes.Structure):
    """Mirror of ``piper_int8_matrix``."""

    _fields_ = [
        ("codes", ctypes.c_void_p),
        ("scale", ctypes.c_void_p),
        ("zero", ctypes.c_void_p),
        ("batch", ctypes.c_int64),
        ("rows", ctypes.c_int64),
        ("cols", ctypes.c_int64),
        ("scale_dtype", ctypes.c_int32),
        ("per_row", ctypes.c_int32),
        ("over_127", ctypes.c_int32),
    ]


class Plan(ctypes.Structure):
    """Mirror of ``piper_int8_plan``."""

    _fields_ = [("tile_tokens", ctypes.c_int32), ("tile_columns", ctypes.c_int32), ("split", ctypes.c_int32),
                ("blocks", ctypes.c_int32)]


_lib = None
_lock = threading.Lock()


def library_path() -> Path:
    return Path(os.environ.get("PIPER_INT8_LIB", LIB_PATH))


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
                f"native INT8 library {path} is missing; build it with "
                "`python -c 'import __graft_entry__ as g; g.build()'` (there is no CPU fallback)."
            )
        lib = ctypes.CDLL(str(path))
        vp, i32, i64, sz = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_size_t
        mat = ctypes.POINTER(Matrix)
        lib.piper_int8_linear_workspace.argtypes = [mat, i64, i32, ctypes.POINTER(sz)]
        lib.piper_int8_grad_input_workspace.argtypes = [mat, i64, i32, ctypes.POINTER(sz)]
        lib.piper_int8_linear.argtypes = [mat, vp, i64, i64, vp, vp, i32, vp, sz, vp]
        lib.piper_int8_grad_input.argtypes = [mat, vp, i64, i64, vp, vp, i32, vp, sz, vp]
        lib.piper_int8_linear_plan.argtypes = [mat, i64, i32, ctypes.POINTER(Plan)]
        lib.piper_int8_grad_input_plan.argtypes = [mat, i64, i32, i32, ctypes.POINTER(Plan)]
        lib.piper_int8_device_status.argtypes = [vp, ctypes.POINTER(ctypes.c_uint32)]
        for name in EXPORTED_SYMBOLS[:6] + ("piper_int8_device_status",):
            getattr(lib, name).restype = ctypes.c_int
        lib.piper_int8_last_error.restype = ctypes.c_char_p
        lib.piper_int8_version.restype = ctypes.c_char_p
        lib.piper_int8_launches.restype = ctypes.c_uint64
        _lib = lib
        return lib


def check(rc: int) -> None:
    if rc == OK:
        return
    msg = load().piper_int8_last_error().decode("utf-8", "replace")
    if rc == EINVAL:
        raise ValueError(msg)
    raise RuntimeError(f"piper int8 failed (status {rc}): {msg}")


def device_status(device: torch.device) -> int:
    """Read and clear the device-side status word (synchronises the current stream)."""
    out = ctypes.c_uint32(0)
    with torch.cuda.device(device):
        rc = load().piper_int8_device_status(current_stream_handle(device), ctypes.byref(out))
    if rc not in (OK, ETIMEOUT):
        check(rc)
    return int(out.value)


def version() -> str:
    return load().piper_int8_version().decode()


def linear_plan(m: Matrix, tokens: int, *, grouped: bool) -> Plan:
    """How the product of a matrix (or a stack of them) and ``tokens`` tokens runs on the current device."""
    plan = Plan()
    check(load().piper_int8_linear_plan(ctypes.byref(m), tokens, grouped, ctypes.byref(plan)))
    return plan


def grad_input_plan(m: Matrix, tokens: int, *, grouped: bool, dtype: int) -> Plan:
    """How the product's gradient runs."""
    plan = Plan()
    check(load().piper_int8_grad_input_plan(ctypes.byref(m), tokens, grouped, dtype, ctypes.byref(plan)))
    return plan


def launches() -> int:
    """Kernels launched by this process through the library so far."""
    return int(load().piper_int8_launches())
