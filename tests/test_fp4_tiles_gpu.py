"""GPU: FP4 products and gradients in each of their tiles, against definitions in 64 bits.

Every case says in which tiles it runs, so that another plan cannot take a kernel out of the tests unseen. Values and
bounds are those of test_fp4_gpu: an fp32 sum is within ``length * 2**-23`` of the sum of magnitudes, a bf16 result
within 2**-8 more of itself. The dense products are made on the device in 64 bits.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import test_fp4_gpu as T
from piper_offload_b200 import _native_fp4 as nat
from piper_offload_b200 import fp4

pytestmark = pytest.mark.gpu

FORMATS, DTYPES = T.FORMATS, T.DTYPES


@pytest.fixture(autouse=True)
def device_status_clean(cuda_device):
    yield
    assert nat.device_status(cuda_device) == 0, "a bounded device wait timed out"


def normal(rows, cols, dtype, device):
    return torch.randn((rows, cols), generator=torch.Generator(device).manual_seed(rows * 7 + cols), device=device).to(dtype)


def dense(a: np.ndarray, device) -> torch.Tensor:
    return torch.from_numpy(a).to(device)


def check(got: torch.Tensor, a: torch.Tensor, b: torch.Tensor) -> None:
    """got = a @ b (64 bits) within the bound."""
    want, size = a @ b, a.abs() @ b.abs()
    bound = size * a.shape[1] * 2.0 ** -23
    if got.dtype is torch.bfloat16:
        bound = bound * (1 + 2.0 ** -8) + want.abs() * 2.0 ** -8
    off = (got.double() - want).abs()
    assert got.isfinite().all()
    assert (off <= bound + 1e-30).all(), f"off by up to {float((off / (bound + 1e-30)).max()):.3g} bounds"


def linear_plan(w, tokens) -> tuple[int, int, int]:
    p = nat.linear_plan(fp4._matrix(w)[0], tokens)
    return p.tile_tokens, p.split, p.fused


def grad_plan(w, tokens, dtype, grouped) -> tuple[int, int, int]:
    p = nat.grad_input_plan(fp4._matrix(w)[0], tokens, grouped=grouped, dtype=fp4._DTYPES[dtype])
    return p.tile_tokens, p.tile_columns, p.split


# ------------------------------------------------------------------------------ products
# several tiles of nine stages for most blocks; one for each; tiles shared by a cluster
LINEAR = [((5000, 1000, 2080), (192, 1, 0)), ((2200, 1500, 2080), (192, 1, 0)), ((3100, 1300, 2080), (128, 1, 0)),
          ((700, 1300, 2080), (128, 1, 0)), ((256, 1100, 16416), (128, 8, 0)), ((600, 1300, 8224), (128, 2, 0)),
          ((180, 2500, 16416), (192, 4, 0))]


@pytest.mark.parametrize("swizzled", [False, True], ids=["rows", "swizzled"])
@pytest.mark.parametrize("shape,plan", LINEAR, ids=lambda v: "x".join(map(str, v)))
@pytest.mark.parametrize("fmt", FORMATS)
def test_products(fmt, shape, plan, swizzled, cuda_device):
    tokens, rows, cols = shape
    w, v = T.make_weight(fmt, rows, cols, cuda_device, swizzled=swizzled, second=0.37 if fmt == "nvfp4" else None)
    assert linear_plan(w, tokens) == plan
    x = normal(tokens, cols, torch.bfloat16, cuda_device)
    check(fp4.linear_fp4(x, w), dense(T.quantized_values(x, fmt), cuda_device), dense(v[0], cuda_device).T)


def test_products_of_columns_that_end_inside_a_step(cuda_device):
    w, v = T.make_weight("nvfp4", 2000, 2064, cuda_device)
    x = normal(3000, 2064, torch.float32, cuda_device)
    assert linear_plan(w, 3000) == (192, 1, 0)
    check(fp4.linear_fp4(x, w), dense(T.quantized_values(x, "nvfp4"), cuda_device), dense(v[0], cuda_device).T)


GROUPED = [((1040, 2080), [900, 0, 1700, 193, 1, 1100], 106, (192, 1, 0)),
           ((1000, 2080), [700, 0, 130, 257, 1, 0, 520, 300, 384, 100], 108, (128, 1, 0)),
           ((700, 1056), [1200, 900, 0, 800, 700, 100, 1000, 1, 700, 599], 0, (192, 1, 0)),
           # more tiles than blocks of the kernel that quantises its tokens: some take a second one
           ((768, 256), [1] * 20 + [80] + [1] * 28, 0, (32, 1, 1)), ((768, 160), [1] * 20 + [70] + [1] * 28, 10, (32, 1, 1))]


@pytest.mark.parametrize("swizzled", [False, True], ids=["rows", "swizzled"])
@pytest.mark.parametrize("shape,sizes,tail,plan", GROUPED, ids=lambda v: "_".join(map(str, v[:6])) if isinstance(v, (list, tuple)) else str(v))
@pytest.mark.parametrize("fmt", FORMATS)
def test_products_by_expert(fmt, shape, sizes, tail, plan, swizzled, cuda_device):
    rows, cols = shape
    tokens = sum(sizes) + tail
    w, v = T.make_weight(fmt, rows, cols, cuda_device, swizzled=swizzled, experts=len(sizes), second=0.5 if fmt == "nvfp4" else None)
    assert linear_plan(w, tokens) == plan
    x = normal(tokens, cols, torch.bfloat16, cuda_device)
    ends = torch.tensor(sizes, device=cuda_device).cumsum(0).to(torch.int32)
    y, xv, at = fp4.grouped_linear_fp4(x, w, ends), dense(T.quantized_values(x, fmt), cuda_device), 0
    for e, n in enumerate(sizes):
        check(y[at:at + n], xv[at:at + n], dense(v[e], cuda_device).T)
        at += n
    assert not y[at:].any()


# ----------------------------------------------------------------------------- gradients
# tiles of 256 columns whose last one ends in its first half (16, 32, 48) or in its second (80, 144, 160, 208)
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("swizzled", [False, True], ids=["rows", "swizzled"])
@pytest.mark.parametrize("fmt,rows,cols", [("nvfp4", 130, 6416), ("nvfp4", 130, 6480), ("nvfp4", 200, 6544), ("nvfp4", 64, 6608),
                                           ("mxfp4", 130, 6432), ("mxfp4", 200, 6560), ("mxfp4", 321, 6656)])
def test_gradients(fmt, rows, cols, swizzled, dtype, cuda_device):
    w, v = T.make_weight(fmt, rows, cols, cuda_device, swizzled=swizzled, second=0.3 if fmt == "nvfp4" else None)
    assert grad_plan(w, 600, dtype, False) == (256, 256, 1)
    dy = normal(600, rows, dtype, cuda_device)
    check(fp4.linear_fp4_grad_input(dy, w), dy.double(), dense(v[0], cuda_device))


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("swizzled", [False, True], ids=["rows", "swizzled"])
@pytest.mark.parametrize("fmt,cols", [("nvfp4", 1296), ("nvfp4", 1424), ("mxfp4", 1312), ("mxfp4", 1440)])
def test_gradients_by_expert(fmt, cols, swizzled, dtype, cuda_device):
    sizes, rows = [300, 0, 40, 1, 0, 90, 60, 0, 65, 7, 0, 130, 17, 0, 2, 110], 130
    tokens = sum(sizes) + 78
    w, v = T.make_weight(fmt, rows, cols, cuda_device, swizzled=swizzled, experts=16, second=0.5 if fmt == "nvfp4" else None)
    assert grad_plan(w, tokens, dtype, True) == (256, 256, 1)
    dy = normal(tokens, rows, dtype, cuda_device)
    ends = torch.tensor(sizes, device=cuda_device).cumsum(0).to(torch.int32)
    dx, at = fp4.grouped_linear_fp4_grad_input(dy, w, ends), 0
    for e, n in enumerate(sizes):
        check(dx[at:at + n], dy[at:at + n].double(), dense(v[e], cuda_device))
        at += n
    assert not dx[at:].any()


@pytest.mark.parametrize("tokens,rows,cols,plan", [(600, 192, 6416, (256, 256, 1)), (300, 200, 256, (256, 128, 1)),
                                                   (40, 4096, 96, (64, 128, 8))])
@pytest.mark.parametrize("fmt", FORMATS)
def test_fp32_gradients_keep_their_last_bits(fmt, tokens, rows, cols, plan, cuda_device):
    """Each column of the weight holds one number, a power of two, so each result is one fp32 value of the gradient
    scaled by it. Adding its three bf16 terms up costs two additions, each within 2**-23; a term less, up to 2**-17."""
    cols = cols // 32 * 32
    g = T.rng(rows, cols)
    at, byte = g.integers(0, rows, cols), 127 if fmt == "mxfp4" else 0x38  # scales of one
    codes = np.zeros((rows, cols), np.uint8)
    codes[at, np.arange(cols)] = g.choice([1, 2, 4, 6, 9, 10, 12, 14], cols)  # 0.5, 1, 2, 4 and the same below zero
    scale = torch.full((rows, cols // T.R.BLOCK[fmt]), byte, dtype=torch.uint8, device=cuda_device)
    q = torch.from_numpy(T.R.pack(codes)).to(cuda_device)
    w = (T.W.MXWeight(q, scale, torch.float4_e2m1fn_x2) if fmt == "mxfp4" else
         T.W.NVFP4Weight(q, scale.view(torch.float8_e4m3fn)))
    assert grad_plan(w, tokens, torch.float32, False) == plan
    dy = normal(tokens, rows, torch.float32, cuda_device)
    value = np.concatenate([T.R.GRID, -T.R.GRID])[codes[at, np.arange(cols)]]
    want = dy[:, torch.from_numpy(at).to(cuda_device)] * torch.from_numpy(value).to(cuda_device, torch.float32)
    off = (fp4.linear_fp4_grad_input(dy, w).double() - want.double()).abs()
    assert (off <= want.double().abs() * 2.0 ** -22).all()


@pytest.mark.parametrize("tokens,rows,cols", [(600, 130, 6416), (5000, 1000, 2080), (3100, 1300, 2080), (180, 2500, 16416)])
@pytest.mark.parametrize("fmt", FORMATS)
def test_repeats_are_bitwise_equal(fmt, tokens, rows, cols, cuda_device):
    w, _ = T.make_weight(fmt, rows, cols // 32 * 32, cuda_device)
    x, dy = (normal(tokens, n, torch.bfloat16, cuda_device) for n in (cols // 32 * 32, rows))
    y, dx = fp4.linear_fp4(x, w), fp4.linear_fp4_grad_input(dy, w)
    for _ in range(4):
        assert torch.equal(fp4.linear_fp4(x, w), y) and torch.equal(fp4.linear_fp4_grad_input(dy, w), dx)
