"""CPU: the INT8 library loads, exports what its header declares, and refuses bad arguments before touching a device; the
reference of the GPU tests is checked against arithmetic in whole numbers."""

from __future__ import annotations

import ctypes
import re
from fractions import Fraction
from pathlib import Path

import numpy as np
import pytest
import torch

import int8_reference as R
from piper_offload_b200 import _native_int8 as nat
from piper_offload_b200 import int8
from piper_offload_b200 import weights as W

HEADER = Path(__file__).resolve().parents[1] / "include" / "piper_int8.h"


def test_library_exports_what_the_header_declares():
    names = set(re.findall(r"\b(piper_int8_\w+)\s*\(", HEADER.read_text()))
    assert names == set(nat.EXPORTED_SYMBOLS)
    for name in names:
        assert hasattr(nat.load(), name), name
    assert "sm_100a" in nat.version()


def matrix(**kw) -> nat.Matrix:
    fields = {"codes": 0x1000, "scale": 0x2000, "zero": None, "batch": 1, "rows": 64, "cols": 96, "scale_dtype": nat.DT_F32,
              "per_row": 1, "over_127": 0}
    return nat.Matrix(**{**fields, **kw})


BAD_MATRICES = [({"rows": 0}, "non-empty"), ({"batch": 0}, "non-empty"), ({"cols": -16}, "non-empty"), ({"cols": nat.MAX_COLS + 1}, "65536"),
                ({"rows": 1 << 31}, "at most"), ({"batch": 1 << 12, "rows": 1 << 20}, "at most"), ({"scale_dtype": 3}, "scales are"),
                ({"batch": 2, "per_row": 0}, "for each row")]


def calls(m: nat.Matrix):
    """Every entry point with arguments that are good but for `m`; none is enqueued when m is bad."""
    lib, ref, n = nat.load(), ctypes.byref(m), ctypes.c_size_t()
    yield lambda: lib.piper_int8_linear_workspace(ref, 8, 1, ctypes.byref(n))
    yield lambda: lib.piper_int8_grad_input_workspace(ref, 8, 0, ctypes.byref(n))
    yield lambda: lib.piper_int8_linear(ref, 0x4000, max(m.cols, 1), 8, 0x5000, 0x6000, 0, 0x100000, 1 << 40, None)
    yield lambda: lib.piper_int8_grad_input(ref, 0x4000, max(m.rows, 1), 8, 0x5000, 0x6000, 0, 0x100000, 1 << 40, None)


@pytest.mark.parametrize("change,match", BAD_MATRICES, ids=lambda v: v if isinstance(v, str) else "-".join(v))
def test_bad_matrices_are_refused(change, match):
    for call in calls(matrix(**change)):
        with pytest.raises(ValueError, match=match):
            nat.check(call())
    with pytest.raises(ValueError, match=match):
        nat.linear_plan(matrix(**change), 8, grouped=True)
    with pytest.raises(ValueError, match=match):
        nat.grad_input_plan(matrix(**change), 8, grouped=True, dtype=0)


@pytest.mark.parametrize("change,match", [({"codes": None}, "null"), ({"scale": None}, "null"), ({"scale": 0x2002}, "aligned")])
def test_bad_buffers_are_refused(change, match):
    for call in list(calls(matrix(**change)))[2:]:  # the workspace queries read no buffers
        with pytest.raises(ValueError, match=match):
            nat.check(call())


@pytest.mark.parametrize("name", ["linear", "grad_input"])
def test_bad_arguments_are_refused(name):
    lib = nat.load()
    function = getattr(lib, f"piper_int8_{name}")

    def call(m=matrix(), **kw):
        a = {"x": 0x4000, "stride": 96, "tokens": 9, "ends": None, "y": 0x6000, "dtype": 0, "ws": 0x100000, "bytes": 1 << 30, **kw}
        return function(ctypes.byref(m), *a.values(), None)

    for kw, match in (({"x": None}, "null"), ({"y": None}, "null"), ({"stride": 63}, "overlap"), ({"tokens": -1}, "tokens"),
                      ({"tokens": 1 << 40}, "tokens"), ({"dtype": 3}, "bfloat16, float16 and float32"), ({"x": 0x4001}, "aligned"),
                      ({"y": 0x6002, "dtype": 2}, "aligned")):
        with pytest.raises(ValueError, match=match):
            nat.check(call(**kw))
    with pytest.raises(ValueError, match="ends"):
        nat.check(call(matrix(batch=3)))
    for kw in ({"ws": None}, {"ws": 0x100010}, {"bytes": 64}):
        with pytest.raises(RuntimeError, match="workspace"):
            nat.check(call(**kw))
    assert call(tokens=0, x=None, y=None) == nat.OK


def test_workspace_needs_are_modest():
    """Aligned codes are used in place: only the tokens need room."""
    lib, n = nat.load(), ctypes.c_size_t()
    m = matrix(rows=4096, cols=4096, codes=1 << 20)
    nat.check(lib.piper_int8_linear_workspace(ctypes.byref(m), 1024, 0, ctypes.byref(n)))
    assert 1024 * 4096 < n.value < 1024 * 4200
    nat.check(lib.piper_int8_grad_input_workspace(ctypes.byref(m), 1024, 0, ctypes.byref(n)))
    assert 2 * 1024 * 4096 < n.value < 2 * 1024 * 4200
    for query in (lambda: lib.piper_int8_linear_workspace(ctypes.byref(m), 0, 0, ctypes.byref(n)),
                  lambda: lib.piper_int8_grad_input_workspace(ctypes.byref(m), 0, 0, ctypes.byref(n))):
        nat.check(query())
        assert n.value == 0


def test_plan_queries():
    """Without a device the plan is made for 148 SMs."""
    for tokens in (1, 40, 700, 5000):
        p = nat.linear_plan(matrix(rows=4096, cols=4096, codes=1 << 20), tokens, grouped=False)
        assert (p.tile_tokens == 8) == (tokens <= 2) and p.tile_tokens in (8, 32, 64, 128, 256) and p.tile_columns in (128, 256) and p.split in (1, 2, 4, 8) and p.blocks in (1, 2)
        p = nat.grad_input_plan(matrix(rows=4096, cols=4096), tokens, grouped=False, dtype=0)
        assert p.tile_tokens in (64, 128, 160, 192, 224, 256) and p.tile_columns in (128, 256, 512)
        assert p.split == 1 or p.tile_columns == 128
        assert p.tile_tokens in (64, 256) or p.tile_columns > 128
    m = matrix()
    for call in (lambda: nat.linear_plan(m, 0, grouped=False), lambda: nat.linear_plan(matrix(batch=2), 8, grouped=False), lambda: nat.grad_input_plan(m, 0, grouped=False, dtype=0),
                 lambda: nat.grad_input_plan(matrix(batch=2), 8, grouped=False, dtype=0)):
        with pytest.raises(ValueError, match="plan query"):
            call()
    with pytest.raises(ValueError, match="bfloat16, float16 and float32"):
        nat.grad_input_plan(m, 8, grouped=False, dtype=4)


def test_cpu_tensors_are_refused():
    x = torch.ones(4, 64, dtype=torch.bfloat16)
    q, s = torch.zeros(8, 64, dtype=torch.int8), torch.ones(8, 1)
    stack = W.Int8Experts(q[None], s[None], (1, 64))
    ends = torch.tensor([4], dtype=torch.int32)
    for call in (lambda: int8.linear_int8(x, W.Int8Weight(q, s, (1, 64))), lambda: int8.linear_int8(x, W.Bnb8Weight(q, s[:, 0])),
                 lambda: int8.linear_int8(x, W.QuantoWeight(q, s, 0, W.QINT8)), lambda: int8.grouped_linear_int8(x, stack, ends),
                 lambda: int8.linear_int8_grad_input(x[:, :8], W.Int8Weight(q, s, (1, 64))),
                 lambda: int8.grouped_linear_int8_grad_input(x[:, :8], stack, ends)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_other_weights_are_refused():
    x = torch.ones(4, 64, dtype=torch.bfloat16)
    gguf = W.GGUFWeight(torch.zeros(8, 68, dtype=torch.uint8), 8)
    fp8 = W.Float8Weight(torch.zeros(8, 64, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.ones(8, 1), (1, 64))
    for call in (lambda w: int8.linear_int8(x, w), lambda w: int8.linear_int8_grad_input(x[:, :8], w)):
        with pytest.raises(ValueError, match="INT8 weights, got GGUFWeight"):
            call(gguf)
        with pytest.raises(ValueError):
            call(fp8)
        with pytest.raises(ValueError):
            call(W.QuantoWeight(fp8.qdata, torch.ones(8, 1), 0, W.QFLOAT8_E4M3))


def test_experts_are_views_of_their_stack():
    stack = W.Int8Experts(torch.zeros(3, 4, 16, dtype=torch.int8), torch.zeros(3, 4, 1), (1, 16), zero_point=torch.zeros(3, 4, 1, dtype=torch.int8))
    assert stack.shape == (3, 4, 16)
    one = stack.expert(1)
    assert one.shape == (4, 16) and one.scale.shape == (4, 1)
    one.qdata.fill_(7)
    one.scale.fill_(5)
    one.zero_point.fill_(3)
    assert stack.qdata[1].eq(7).all() and not stack.qdata[0].any() and stack.scale[1].eq(5).all() and not stack.scale[2].any()
    assert stack.zero_point[1].eq(3).all() and not stack.zero_point[0].any()


# ------------------------------------------------- the reference against whole numbers
def test_reference_codes_are_of_the_exact_quotient():
    g = np.random.default_rng(1)
    x = g.standard_normal((20, 64)).astype(np.float32).astype(np.float64)
    top = np.abs(x).max(axis=1, keepdims=True)
    x[:, 1::2] = ((np.arange(32) * 4 + 0.5)[None, :] * top / 127).astype(np.float32)
    x[0] = 0
    x[1, :] = 3 * 2.0 ** -149
    x[2] = np.arange(64) - 63.5
    x[2, 0] = 127
    codes, scale = R.quantize(x)
    for i in range(20):
        a = max(abs(Fraction(v)) for v in x[i])
        for j in range(64):
            want = 0 if a == 0 else round(127 * Fraction(x[i, j]) / a)  # a Fraction rounds half to even
            assert codes[i, j] == want
        assert scale[i, 0] == np.abs(x[i]).max() / 127
