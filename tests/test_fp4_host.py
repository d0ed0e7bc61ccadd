"""CPU: the FP4 library loads, exports what its header declares, and refuses bad arguments before touching a device;
the reference the GPU tests compare with is checked against the merges' oracle."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import numpy as np
import pytest
import torch

import fp4_reference as R
from oracle import numerics as N
from piper_offload_b200 import _native_fp4 as nat
from piper_offload_b200 import fp4
from piper_offload_b200 import weights as W

HEADER = Path(__file__).resolve().parents[1] / "include" / "piper_fp4.h"


def test_library_exports_what_the_header_declares():
    names = set(re.findall(r"\b(piper_fp4_\w+)\s*\(", HEADER.read_text()))
    assert names == set(nat.EXPORTED_SYMBOLS)
    for name in names:
        assert hasattr(nat.load(), name), name
    assert "sm_100a" in nat.version()


def matrix(**kw) -> nat.Matrix:
    fields = {"codes": 0x1000, "scale": 0x2000, "second": None, "batch": 1, "rows": 64, "cols": 96, "format": nat.FMT_NV,
              "swizzled": 1}
    return nat.Matrix(**{**fields, **kw})


BAD_MATRICES = [({"format": 7}, "unknown format"), ({"rows": 0}, "non-empty"), ({"batch": 0}, "non-empty"),
                ({"cols": 40}, "divisible by 16"), ({"cols": 48, "format": nat.FMT_MX}, "divisible by 32"),
                ({"rows": 1 << 31}, "at most"), ({"batch": 1 << 12, "rows": 1 << 20}, "at most"),
                ({"second": 0x3000, "format": nat.FMT_MX}, "no second-level")]


def calls(m: nat.Matrix):
    """Every entry point with arguments that are good but for `m`; none is enqueued when m is bad."""
    lib, ref, n = nat.load(), ctypes.byref(m), ctypes.c_size_t()
    yield lambda: lib.piper_fp4_quantize(ref, 0x4000, m.cols, 0, 0, 0, None, None)
    yield lambda: lib.piper_fp4_dequantize(ref, 0x4000, 0, None)
    yield lambda: lib.piper_fp4_linear_workspace(ref, 8, ctypes.byref(n))
    yield lambda: lib.piper_fp4_grad_input_workspace(ref, 0x4000, m.rows, 8, 0, ctypes.byref(n))
    yield lambda: lib.piper_fp4_linear(ref, 0x4000, m.cols, 8, 0x5000, None, 0, 0x6000, 0, 0x100000, 1 << 30, None)
    yield lambda: lib.piper_fp4_grad_input(ref, 0x4000, m.rows, 8, 0x5000, 0x6000, 0, None, 0, None)


@pytest.mark.parametrize("change,match", BAD_MATRICES, ids=lambda v: v if isinstance(v, str) else "-".join(v))
def test_bad_matrices_are_refused(change, match):
    for call in calls(matrix(**change)):
        with pytest.raises(ValueError, match=match):
            nat.check(call())


@pytest.mark.parametrize("change", [{"codes": None}, {"scale": None}])
def test_null_buffers_are_refused(change):
    m = matrix(**change)
    for i, call in enumerate(calls(m)):
        if i not in (2, 3):  # the workspace queries read no buffers
            with pytest.raises(ValueError, match="null"):
                nat.check(call())


def test_bad_arguments_are_refused():
    lib, m = nat.load(), matrix()
    ref = ctypes.byref(m)

    def linear(**kw):
        a = {"x": 0x4000, "stride": 96, "tokens": 8, "ends": None, "act": None, "mode": 0, "y": 0x6000, "dtype": 0,
             "ws": 0x100000, "bytes": 1 << 30, **kw}
        return lib.piper_fp4_linear(a.pop("ref", ref), *a.values(), None)

    for kw, match in (({"x": None}, "null"), ({"y": None}, "null"), ({"stride": 95}, "overlap"), ({"tokens": -1}, "tokens"),
                      ({"tokens": 1 << 40}, "tokens"), ({"mode": 4}, "scaling mode"), ({"dtype": 1}, "bfloat16 and float32")):
        with pytest.raises(ValueError, match=match):
            nat.check(linear(**kw))
    for kw in ({"ws": None}, {"ws": 0x100010}, {"bytes": 64}):  # many tokens are quantized into it
        with pytest.raises(RuntimeError, match="workspace"):
            nat.check(linear(tokens=800, **kw))
    assert linear(tokens=0, x=None, y=None) == nat.OK

    several = matrix(batch=3)
    with pytest.raises(ValueError, match="ends"):
        nat.check(lib.piper_fp4_linear(ctypes.byref(several), 0x4000, 96, 8, None, None, 0, 0x6000, 0, 0x100000, 1 << 30, None))
    with pytest.raises(ValueError, match="ends"):
        nat.check(lib.piper_fp4_grad_input(ctypes.byref(several), 0x4000, 64, 8, None, 0x6000, 0, None, 0, None))
    mx = matrix(format=nat.FMT_MX)
    with pytest.raises(ValueError, match="no second-level"):
        nat.check(lib.piper_fp4_linear(ctypes.byref(mx), 0x4000, 96, 8, None, 0x7000, 0, 0x6000, 0, 0x100000, 1 << 30, None))
    with pytest.raises(RuntimeError, match="workspace"):  # fp32 gradients are split in a workspace
        nat.check(lib.piper_fp4_grad_input(ref, 0x4000, 64, 8, None, 0x6000, 2, None, 0, None))

    def quantize(m, **kw):
        a = {"x": 0x4000, "stride": 96, "dtype": 0, "mode": 0, "second": 0, "maxima": None, **kw}
        return lib.piper_fp4_quantize(ctypes.byref(m), *a.values(), None)

    for m2, kw, match in ((m, {"x": None}, "null"), (m, {"stride": 64}, "overlap"), (m, {"dtype": 1}, "bfloat16"),
                          (m, {"mode": 9}, "scaling mode"), (m, {"second": 3}, "second-level mode"), (m, {"second": 1}, "match"),
                          (matrix(second=0x3000), {}, "match"), (matrix(second=0x3000, rows=4096), {"second": 2}, "maxima"),
                          (matrix(codes=0x1002), {}, "4-byte")):
        with pytest.raises(ValueError, match=match):
            nat.check(quantize(m2, **kw))


def test_workspace_needs_are_modest():
    """Aligned swizzled weights are used in place: only the tokens' codes and scales need room."""
    lib, n = nat.load(), ctypes.c_size_t()
    m = matrix(rows=4096, cols=4096, codes=1 << 20, scale=1 << 20)
    nat.check(lib.piper_fp4_linear_workspace(ctypes.byref(m), 1024, ctypes.byref(n)))
    assert n.value < 1024 * 4096
    nat.check(lib.piper_fp4_grad_input_workspace(ctypes.byref(m), 1 << 20, 4096, 1024, 0, ctypes.byref(n)))
    assert n.value == 0


def test_cpu_tensors_are_refused():
    x = torch.ones(4, 64, dtype=torch.bfloat16)
    q, s = torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 4, dtype=torch.uint8).view(torch.float8_e4m3fn)
    for call in (lambda: fp4.quantize_mxfp4(x), lambda: fp4.quantize_nvfp4(x), lambda: fp4.dequantize_fp4(W.NVFP4Weight(q, s)),
                 lambda: fp4.linear_fp4(x, W.NVFP4Weight(q, s)), lambda: fp4.linear_fp4_grad_input(x[:, :8], W.NVFP4Weight(q, s))):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_other_weights_are_refused():
    x = torch.ones(4, 64, dtype=torch.bfloat16)
    gguf = W.GGUFWeight(torch.zeros(8, 68, dtype=torch.uint8), 8)
    fp8 = W.Float8Weight(torch.zeros(8, 64, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.ones(8, 1), (1, 64))
    for call in (lambda w: fp4.linear_fp4(x, w), lambda w: fp4.linear_fp4_grad_input(x[:, :8], w), fp4.dequantize_fp4):
        with pytest.raises(ValueError, match="MXFP4 and NVFP4 weights, got GGUFWeight"):
            call(gguf)
        with pytest.raises(ValueError):
            call(fp8)


def test_experts_are_views_of_their_stack():
    stack = W.NVFP4Experts(torch.zeros(3, 4, 16, dtype=torch.uint8), torch.zeros(3, 4, 2, dtype=torch.uint8),
                           torch.ones(3), is_swizzled_scales=False)
    assert stack.shape == (3, 4, 32)
    one = stack.expert(1)
    assert one.shape == (4, 32)
    one.qdata.fill_(7)
    one.scale.fill_(5)
    one.per_tensor_scale.fill_(3)
    assert stack.qdata[1].eq(7).all() and not stack.qdata[0].any() and stack.scale[1].eq(5).all()
    assert stack.per_tensor_scale.tolist() == [1, 3, 1]
    mx = W.MXExperts(torch.zeros(2, 4, 16, dtype=torch.uint8), torch.zeros(2, 4, 1, dtype=torch.uint8), torch.float4_e2m1fn_x2)
    assert mx.shape == (2, 4, 32) and mx.expert(1).shape == (4, 32)


# ------------------------------------------------- the reference against the oracle
def test_reference_codecs_agree_with_the_oracle():
    x = np.concatenate([np.linspace(-7, 7, 4001), R.GRID, -R.GRID, (R.GRID[1:] + R.GRID[:-1]) / 2]).astype(np.float32)
    np.testing.assert_array_equal(R.encode_e2m1(x.astype(np.float64)), N.encode_e2m1(np.clip(x, -6, 6)))
    s = np.concatenate([np.linspace(0.015625, 448, 20001), R.E4M3[:127], (R.E4M3[1:127] + R.E4M3[:126]) / 2]).astype(np.float32)
    np.testing.assert_array_equal(R.encode_e4m3(s.astype(np.float64)), N.encode_e4m3(s))
    codes = np.arange(256, dtype=np.uint8)
    np.testing.assert_array_equal(R.E4M3.astype(np.float32), N.decode_e4m3(codes))


@pytest.mark.parametrize("mode", ["floor", "rceil", "ceil", "even"])
def test_reference_quantisation_is_the_merges_encoder(mode):
    """A merge of nothing into exactly held values re-encodes them as the quantiser does."""
    from oracle import merge as M

    g = np.random.default_rng(3)
    x = g.standard_normal((32, 256)).astype(np.float32)
    codes, byte = R.quantize(x.astype(np.float64), "mxfp4", mode=mode)
    target, limit, bits = M.MX_FORMATS["e2m1"]
    want, inverse = M.mx_calculate_scale(np.abs(x).reshape(32, 8, 32).max(-1), target, limit, bits, M.MX_SCALE_MODES[mode])
    np.testing.assert_array_equal(byte, want)
    np.testing.assert_array_equal(codes, N.encode_e2m1(np.clip(x * np.repeat(inverse, 32, axis=1), -6, 6)))


def test_reference_places_are_the_oracles():
    from oracle import merge as M

    for rows, blocks in ((1, 1), (70, 13), (128, 4), (300, 9)):
        for swizzled in (False, True):
            np.testing.assert_array_equal(R.scale_places(rows, blocks, swizzled), M.scale_index(rows, blocks, swizzled))


# ------------------------------------------------------------------------ plans
def test_plan_queries():
    """Without a device the plan is made for 148 SMs."""
    def linear(tokens, **kw):
        p = nat.linear_plan(matrix(**kw), tokens)
        return p.tile_tokens, p.tile_columns, p.split, p.fused

    def grad(tokens, dtype=nat.DT_BF16, **kw):
        p = nat.grad_input_plan(matrix(**kw), tokens, grouped=kw.get("batch", 1) > 1, dtype=dtype)
        return p.tile_tokens, p.tile_columns, p.split, p.fused

    for tokens in (1, 40, 700, 5000):
        tile, columns, split, fused = linear(tokens, rows=4096, cols=4096)
        assert tile in (32, 128, 192) and columns == 128 and split in (1, 2, 4, 8) and fused == (tokens <= 2)
        tile, columns, split, fused = grad(tokens, rows=4096, cols=4096)
        assert tile in (64, 256) and columns in (128, 256) and not fused
        assert split == 1 or columns == 128
    # sums of groups, whose tiles are found on the device, and of wide tiles are not shared
    assert linear(64, batch=8, rows=128, cols=8192)[2] == grad(64, batch=8, rows=8192, cols=128)[2] == 1
    m = matrix()
    for call in (lambda: nat.linear_plan(m, 0), lambda: nat.grad_input_plan(m, 0, grouped=False, dtype=0),
                 lambda: nat.grad_input_plan(matrix(batch=2), 8, grouped=False, dtype=0)):
        with pytest.raises(ValueError, match="plan query"):
            call()
    with pytest.raises(ValueError, match="bfloat16 and float32"):
        nat.grad_input_plan(m, 8, grouped=False, dtype=1)
    for change, match in BAD_MATRICES:
        with pytest.raises(ValueError, match=match):
            nat.linear_plan(matrix(**change), 8)
        with pytest.raises(ValueError, match=match):
            nat.grad_input_plan(matrix(**change), 8, grouped=True, dtype=0)
