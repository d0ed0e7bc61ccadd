"""GPU: INT8 products and gradients in each of their tiles, against definitions in 64 bits.

Every case says in which tiles it runs, so that another plan cannot take a kernel out of the tests unseen. Bounds are
those of int8_reference; the dense products are made on the device in 64 bits, where sums of codes are exact.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import int8_reference as R
import test_int8_gpu as T
from piper_offload_b200 import _native_int8 as nat
from piper_offload_b200 import int8
from piper_offload_b200 import weights as W

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def device_status_clean(cuda_device):
    yield
    assert nat.device_status(cuda_device) == 0, "a bounded device wait timed out"


def made(batch, rows, cols, device, seed=0):
    """An asymmetric stack of experts, or one weight, its codes less zero points and its scales in 64 bits."""
    g = torch.Generator(device).manual_seed(seed)
    q = torch.randint(-128, 128, (batch, rows, cols), generator=g, device=device, dtype=torch.int16).to(torch.int8)
    z = torch.randint(-128, 128, (batch, rows, 1), generator=g, device=device, dtype=torch.int16).to(torch.int8)
    s = (torch.rand((batch, rows, 1), generator=g, device=device) * 0.01 + 1e-4).bfloat16()
    values, scale = q.double() - z.double(), s.double()[..., 0]
    if batch == 1:
        return W.Int8Weight(q[0], s[0], (1, cols), zero_point=z[0]), values, scale
    return W.Int8Experts(q, s, (1, cols), zero_point=z), values, scale


def ends_of(batch, tokens, device) -> torch.Tensor:
    """Uneven groups, one of them empty, the last rows no expert's."""
    share = np.array([3, 1, 0, 5, 2, 4][:batch], float)
    return torch.tensor(np.cumsum(share / share.sum() * (tokens - tokens // 50)).astype(np.int32), device=device)


def quantized(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales of tokens whose quotients are no closer to a half than fp64 tells apart: 16-bit values are not."""
    a = x.double().abs().amax(1, keepdim=True)
    return torch.round(x.double() * 127 / a), a / 127


def check_product(y, x, values, scale, ends) -> None:
    q, s = quantized(x)
    at = 0
    for e, end in enumerate(ends):
        want = (q[at:end] @ values[e].T) * s[at:end] * scale[e][None, :]
        off, bound = (y[at:end].double() - want).abs(), want.abs() * (5 * 2.0 ** -24 + R.EPS[T.name(x.dtype)]) * (1 + 2.0 ** -7) + R.TINY[T.name(x.dtype)]
        assert (off <= bound).all(), f"off by up to {float((off / bound).max()):.3g} bounds"
        at = end
    assert not y[at:].any()


def check_gradient(dx, dy, values, scale, ends) -> None:
    at, dtype = 0, T.name(dy.dtype)
    terms = 2 if dy.dtype is torch.float32 else 1
    for e, end in enumerate(ends):
        v = dy[at:end].double() * scale[e][None, :]
        if end > at:
            want, size = v @ values[e], v.abs() @ values[e].abs()
            bound = size * (2.0 ** (-11 * terms) + 2 * 2.0 ** -24 + terms * values.shape[1] * 2.0 ** -23)
            bound += v.abs().amax(1, keepdim=True) * 2.0 ** -39 * values[e].abs().sum(0)[None, :]
            bound = bound * (1 + 2.0 ** -7) + want.abs() * R.EPS[dtype] + R.TINY[dtype]
            off = (dx[at:end].double() - want).abs()
            assert (off <= bound).all(), f"off by up to {float((off / bound).max()):.3g} bounds"
        at = end
    assert not dx[at:].any()


# (batch, tokens, rows, cols), (tile of tokens, of outputs, blocks that share sums, blocks an SM)
LINEAR = [((1, 1, 14336, 1040), (8, 128, 1, 1)), ((1, 3, 200, 1040), (8, 128, 2, 1)), ((1, 4, 200, 2000), (8, 128, 4, 1)),
          ((1, 2, 200, 4096), (8, 128, 8, 1)), ((1, 8, 130, 1024), (8, 128, 2, 1)), ((1, 8, 200, 1040), (32, 128, 1, 1)),
          ((1, 1, 20000, 1040), (32, 128, 1, 2)), ((1, 150, 1000, 4096), (32, 128, 2, 2)), ((1, 100, 600, 2320), (32, 128, 4, 2)),
          ((1, 8, 200, 2000), (32, 128, 8, 2)), ((1, 200, 3000, 1040), (64, 128, 1, 1)), ((1, 40, 20000, 1040), (64, 128, 1, 2)),
          ((1, 300, 1000, 8000), (64, 128, 2, 1)), ((1, 40, 3000, 4096), (64, 128, 4, 1)), ((1, 40, 2000, 4096), (64, 128, 8, 1)),
          ((1, 200, 5000, 1040), (128, 128, 1, 1)), ((1, 70, 3000, 8000), (128, 128, 4, 1)), ((1, 70, 2000, 4096), (128, 128, 8, 1)),
          ((1, 300, 2000, 1040), (128, 256, 1, 1)), ((1, 150, 14336, 1040), (256, 128, 1, 1)), ((1, 150, 2000, 8000), (256, 128, 8, 1)),
          ((1, 500, 5000, 1040), (256, 256, 1, 1)), ((1, 2100, 5000, 1100), (256, 256, 1, 1)),
          ((6, 50, 200, 1040), (32, 128, 1, 1)), ((6, 8, 5000, 1040), (32, 128, 1, 2)), ((6, 1000, 600, 1040), (64, 128, 1, 1)),
          ((6, 1000, 2000, 1040), (64, 128, 1, 2)), ((6, 500, 2000, 1040), (128, 128, 1, 1)), ((6, 5000, 200, 1040), (128, 256, 1, 1)),
          ((6, 1500, 2000, 1040), (256, 128, 1, 1)), ((6, 5000, 333, 1040), (256, 256, 1, 1))]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("shape,tile", LINEAR, ids=lambda v: "-".join(map(str, v)))
def test_product_tiles(shape, tile, dtype, cuda_device):
    batch, tokens, rows, cols = shape
    w, values, scale = made(batch, rows, cols, cuda_device)
    plan = nat.linear_plan(int8._Frozen(w, 2 if batch == 1 else 3).matrix, tokens, grouped=batch > 1)
    assert (plan.tile_tokens, plan.tile_columns, plan.split, plan.blocks) == tile
    x = torch.randn((tokens, cols), generator=torch.Generator(cuda_device).manual_seed(1), device=cuda_device).to(dtype)
    if batch == 1:
        check_product(int8.linear_int8(x, w), x, values, scale, [tokens])
        # more than one weight's worth of blocks at once: another call under way on another stream
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = int8.linear_int8(x, w)
        mine = int8.linear_int8(x, w)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(mine, other)
    else:
        ends = ends_of(batch, tokens, cuda_device)
        check_product(int8.grouped_linear_int8(x, w, ends), x, values, scale, ends.tolist())


# (batch, tokens, rows, cols), (tile of tokens, of columns, blocks that share sums)
GRAD = [((1, 20, 520, 100), (64, 128, 1)), ((1, 9, 1000, 9000), (64, 128, 2)), ((1, 7, 520, 100), (64, 128, 4)), ((1, 48, 1000, 100), (64, 128, 8)),
        ((1, 300, 520, 100), (192, 256, 1)), ((1, 1500, 520, 4096), (192, 512, 1)), ((1, 70, 520, 100), (256, 128, 1)),
        ((1, 70, 2050, 9000), (256, 128, 2)), ((1, 70, 2050, 4096), (256, 128, 4)), ((1, 70, 1100, 100), (256, 128, 8)),
        ((1, 1000, 520, 4096), (256, 256, 1)), ((1, 70, 520, 20000), (256, 512, 1)), ((1, 1000, 520, 20000), (224, 512, 1)),
        ((6, 250, 520, 100), (64, 128, 1)), ((6, 1500, 520, 100), (192, 256, 1)), ((6, 3000, 520, 2048), (192, 512, 1)),
        ((6, 1500, 520, 2048), (224, 256, 1)), ((6, 1500, 520, 4096), (224, 512, 1)), ((6, 300, 520, 100), (256, 128, 1)),
        ((6, 1000, 520, 100), (256, 256, 1)), ((6, 300, 520, 4096), (256, 512, 1))]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("shape,tile", GRAD, ids=lambda v: "-".join(map(str, v)))
def test_gradient_tiles(shape, tile, dtype, cuda_device):
    batch, tokens, rows, cols = shape
    w, values, scale = made(batch, rows, cols, cuda_device)
    plan = nat.grad_input_plan(int8._Frozen(w, 2 if batch == 1 else 3).matrix, tokens, grouped=batch > 1, dtype=int8._DTYPES[dtype])
    assert (plan.tile_tokens, plan.tile_columns, plan.split) == tile
    dy = torch.randn((tokens, rows), generator=torch.Generator(cuda_device).manual_seed(1), device=cuda_device).to(dtype)
    if batch == 1:
        check_gradient(int8.linear_int8_grad_input(dy, w), dy, values, scale, [tokens])
    else:
        ends = ends_of(batch, tokens, cuda_device)
        check_gradient(int8.grouped_linear_int8_grad_input(dy, w, ends), dy, values, scale, ends.tolist())


@pytest.mark.parametrize("tokens,rows,cols", [(600, 300, 1100), (2100, 1000, 520), (3, 130, 260)])
def test_fp32_in_wide_tiles(tokens, rows, cols, cuda_device):
    w, values, scale = made(1, rows, cols, cuda_device)
    x = torch.randn((tokens, cols), generator=torch.Generator(cuda_device).manual_seed(1), device=cuda_device)
    q = torch.from_numpy(R.quantize(x.double().cpu().numpy())[0]).to(cuda_device)
    s = x.double().abs().amax(1, keepdim=True) / 127
    want = (q @ values[0].T) * s * scale[0][None, :]
    assert ((int8.linear_int8(x, w).double() - want).abs() <= want.abs() * 5.1 * 2.0 ** -24).all()
    dy = torch.randn((tokens, rows), generator=torch.Generator(cuda_device).manual_seed(2), device=cuda_device)
    check_gradient(int8.linear_int8_grad_input(dy, w), dy, values, scale, [tokens])


def test_offsets_beyond_32_bits(cuda_device):
    """Codes, tokens and results that end more than 2^32 bytes into their tensors."""
    rows, cols = 40000, 40000  # 1.6 GB an expert
    if torch.cuda.get_device_properties(cuda_device).total_memory < 60e9:
        pytest.skip("needs 20 GB")
    q = torch.empty((3, rows, cols), dtype=torch.int8, device=cuda_device)
    for e in range(3):
        q[e].random_(-127, 128, generator=torch.Generator(cuda_device).manual_seed(e))
    s = torch.full((3, rows, 1), 2.0 ** -10, device=cuda_device, dtype=torch.bfloat16)
    w = W.Int8Experts(q, s, (1, cols))
    ends = torch.tensor([2, 2, 5], dtype=torch.int32, device=cuda_device)
    x = torch.randn((5, cols), generator=torch.Generator(cuda_device).manual_seed(1), device=cuda_device).bfloat16()
    y = int8.grouped_linear_int8(x, w, ends)
    dx = int8.grouped_linear_int8_grad_input(y, w, ends)
    codes, unit = quantized(x)
    at = slice(rows - 300, rows)
    check_product(y[2:, at], x[2:], q[2:, at].double(), s.double()[2:, at, 0], [3])
    want, size = torch.zeros((3, 64), dtype=torch.float64, device=cuda_device), torch.zeros((3, 64), dtype=torch.float64, device=cuda_device)
    v = y[2:].double() * 2.0 ** -10
    want += v @ q[2, :, -64:].double()
    size += v.abs() @ q[2, :, -64:].double().abs()
    bound = size * (2.0 ** -11 + 2 * 2.0 ** -24 + rows * 2.0 ** -23) + want.abs() * 2.0 ** -8
    assert ((dx[2:, -64:].double() - want).abs() <= bound).all()
    del q, s, w, y, dx
    torch.cuda.empty_cache()
    # many rows: results past 2^32 bytes
    tokens, rows, cols = 150000, 16400, 64
    w, values, scale = made(1, rows, cols, cuda_device)
    x = torch.randn((tokens, cols), generator=torch.Generator(cuda_device).manual_seed(1), device=cuda_device).bfloat16()
    y = int8.linear_int8(x, w)
    check_product(y[-200:], x[-200:], values, scale, [200])
    dx = int8.linear_int8_grad_input(y, w)
    check_gradient(dx[-200:], y[-200:], values, scale, [200])
