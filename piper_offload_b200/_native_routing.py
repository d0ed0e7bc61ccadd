"""ctypes binding of ``libpiper_routing.so`` (the sm_100a C ABI in ``include/piper_routing.h``).

As with the merges there is no fallback: a missing library raises
``RuntimeError`` at the first call.
"""

from __future__ import annotations

import ctypes
import os
import threading
from pathlib import Path

from ._native import EINVAL, OK

LIB_PATH = Path(__file__).resolve().parent / "libpiper_routing.so"

DT_BF16 = 0
DT_F16 = 1
DT_F32 = 2
SOFTMAX = 0
SIGMOID = 1
MAX = 0
TOP2 = 1
MAX_EXPERTS = 1024  # PIPER_ROUTING_MAX_EXPERTS
MAX_TOP_K = 32  # PIPER_ROUTING_MAX_TOP_K
MAX_GROUPS = 32  # PIPER_ROUTING_MAX_GROUPS

EXPORTED_SYMBOLS = (
    "piper_routing_workspace",
    "piper_routing_route",
    "piper_routing_route_grad",
    "piper_routing_dispatch",
    "piper_routing_combine",
    "piper_routing_combine_grad",
    "piper_routing_last_error",
    "piper_routing_version",
    "piper_routing_launches",
)


class Config(ctypes.Structure):
    """Mirror of ``piper_routing_config``."""

    _fields_ = [
        ("tokens", ctypes.c_int64),
        ("experts", ctypes.c_int32),
        ("top_k", ctypes.c_int32),
        ("scoring", ctypes.c_int32),
        ("groups", ctypes.c_int32),
        ("top_groups", ctypes.c_int32),
        ("group_score", ctypes.c_int32),
        ("renormalize", ctypes.c_int32),
        ("scale", ctypes.c_float),
    ]


class Exchange(ctypes.Structure):
    """Mirror of ``piper_routing_exchange``."""

    _fields_ = [
        ("tokens", ctypes.c_int64),
        ("top_k", ctypes.c_int32),
        ("hidden", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("rows", ctypes.c_void_p),
        ("total", ctypes.c_void_p),
    ]


_lib = None
_lock = threading.Lock()


def library_path() -> Path:
    return Path(os.environ.get("PIPER_ROUTING_LIB", LIB_PATH))


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
                f"native routing library {path} is missing; build it with "
                "`python -c 'import __graft_entry__ as g; g.build()'` (there is no CPU fallback)."
            )
        lib = ctypes.CDLL(str(path))
        vp, i32, i64, sz = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_size_t
        cfg, ex = ctypes.POINTER(Config), ctypes.POINTER(Exchange)
        lib.piper_routing_workspace.argtypes = [cfg, ctypes.POINTER(sz)]
        lib.piper_routing_route.argtypes = [cfg, vp, i64, i32, vp, vp, vp, vp, vp, vp, vp, vp, sz, vp]
        lib.piper_routing_route_grad.argtypes = [cfg, vp, i64, i32, vp, vp, vp, vp]
        lib.piper_routing_dispatch.argtypes = [ex, vp, i64, vp, vp]
        lib.piper_routing_combine.argtypes = [ex, vp, i64, vp, vp, vp]
        lib.piper_routing_combine_grad.argtypes = [ex, vp, i64, vp, vp, i64, vp, vp, vp]
        for name in EXPORTED_SYMBOLS[:6]:
            getattr(lib, name).restype = ctypes.c_int
        lib.piper_routing_last_error.restype = ctypes.c_char_p
        lib.piper_routing_version.restype = ctypes.c_char_p
        lib.piper_routing_launches.restype = ctypes.c_uint64
        _lib = lib
        return lib


def check(rc: int) -> None:
    if rc == OK:
        return
    msg = load().piper_routing_last_error().decode("utf-8", "replace")
    if rc == EINVAL:
        raise ValueError(msg)
    raise RuntimeError(f"piper routing failed (status {rc}): {msg}")


def version() -> str:
    return load().piper_routing_version().decode()


def launches() -> int:
    """Kernels launched by this process through the library so far."""
    return int(load().piper_routing_launches())
