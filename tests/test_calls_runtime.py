"""The compiled calls share the process's C++ runtime: a library call that fails raises its message."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

from piper_offload_b200 import build

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.parametrize("out", [build.CALLS_OUT, build.EXPERT_CALLS_OUT], ids=lambda p: p.stem)
def test_no_second_runtime(out):
    """The output stream's number formatting comes from outside, if at all."""
    if not out.exists():
        build.build()
    defined = subprocess.run(["nm", "-D", "--defined-only", str(out)], check=True, capture_output=True, text=True).stdout
    assert "_ZNSo" not in defined and "_ZNSt6locale" not in defined


# in a process of its own, which the error may not end
FAILS = """
import ctypes
import torch
from piper_offload_b200 import _native_calls, int8, routing, weights

calls = _native_calls.calls()
status = ctypes.CFUNCTYPE(ctypes.c_int)(lambda: {status})
message = ctypes.CFUNCTYPE(ctypes.c_void_p)(lambda: ctypes.cast(text, ctypes.c_void_p).value)
text = ctypes.c_char_p(b"what went wrong")
here, told = (ctypes.cast(f, ctypes.c_void_p).value for f in (status, message))
calls.bind(*[here] * 4, told, *[here] * 6, told)
x = torch.ones(4, 64, device="cuda")
w = weights.Int8Weight(torch.ones(32, 64, dtype=torch.int8, device="cuda"), torch.ones(32, 1, device="cuda"), (1, 64))
r = routing.Routing(x[:, :2].contiguous(), *(torch.zeros(4, 2, dtype=torch.int32, device="cuda") for _ in range(3)), None)
r.ends = r.ends[0]
for call in (lambda: int8.linear_int8(x, w), lambda: int8.linear_int8(x.clone().requires_grad_(), w),
             lambda: routing.route_tokens(x, 2), lambda: routing.dispatch_tokens(x, r)):
    try:
        call()
    except {error} as exc:
        print(str(exc).splitlines()[0])
"""


@pytest.mark.gpu
@pytest.mark.parametrize("status,error,told", [(2, "RuntimeError", "piper {} failed (status 2): what went wrong"), (1, "ValueError", "what went wrong")])
def test_a_failed_call_raises(status, error, told, cuda_device):
    done = subprocess.run([sys.executable, "-c", FAILS.format(status=status, error=error)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
    assert done.stdout.splitlines() == [told.format(name) for name in ("int8", "int8", "routing", "routing")]
