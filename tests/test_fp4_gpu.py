"""GPU: the FP4 operators against their definitions in 64 bits (fp4_reference).

Quantisation is compared code for code and byte for byte. Products of bf16
tokens round an fp32 sum once: the result is within 2**-8 of the value, plus
the sum's own error, at most ``cols * 2**-23`` of the sum of magnitudes (every
product of two e2m1 codes and two scales is exact in fp32). fp32 results are
held to that second bound alone, gradients with ``rows`` in its place.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import fp4_reference as R
from piper_offload_b200 import _native_fp4 as nat
from piper_offload_b200 import fp4
from piper_offload_b200 import weights as W

pytestmark = pytest.mark.gpu

FORMATS = ["mxfp4", "nvfp4"]
MODES = ["floor", "rceil", "ceil", "even"]
DTYPES = [torch.bfloat16, torch.float32]


@pytest.fixture(autouse=True)
def device_status_clean(cuda_device):
    yield
    assert nat.device_status(cuda_device) == 0, "a bounded device wait timed out"


def rng(*key: int) -> np.random.Generator:
    return np.random.default_rng(list(key))


def to_torch(x: np.ndarray, dtype, device) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(x)).to(device=device, dtype=dtype)


def exact(t: torch.Tensor) -> np.ndarray:
    return t.detach().double().cpu().numpy()


def codes_of(w) -> np.ndarray:
    return R.unpack(w.qdata.cpu().numpy())


def bytes_of(w) -> np.ndarray:
    return w.scale.view(torch.uint8).cpu().numpy()


def make_weight(fmt, rows, cols, device, *, seed=0, swizzled=True, second=None, experts=None, padding=0, dtype=torch.bfloat16):
    """A packed weight (or stack) of random codes and scales, and its values (experts, rows, cols)."""
    g = rng(seed, rows, cols)
    e = experts or 1
    codes = g.integers(0, 16, (e, rows, cols), dtype=np.uint8)
    blocks = cols // R.BLOCK[fmt]
    if fmt == "mxfp4":
        byte = g.integers(118, 126, (e, rows, blocks)).astype(np.uint8)
    else:
        byte = g.integers(24, 72, (e, rows, blocks)).astype(np.uint8)
    s2 = None if second is None else np.float32(second) * (1 + np.arange(e, dtype=np.float32))
    value = np.stack([R.values(codes[i], byte[i], fmt, None if s2 is None else s2[i]) for i in range(e)])
    scale = np.stack([R.lay_out(byte[i], swizzled, padding) for i in range(e)])
    q = torch.from_numpy(R.pack(codes)).to(device)
    s = torch.from_numpy(scale).to(device)
    if not experts:
        q, s = q[0].contiguous(), s[0].contiguous()
    t2 = None if s2 is None else torch.from_numpy(s2).to(device)
    if fmt == "mxfp4":
        kind = W.MXExperts if experts else W.MXWeight
        return kind(q, s, torch.float4_e2m1fn_x2, orig_dtype=dtype, is_swizzled_scales=swizzled), value
    kind = W.NVFP4Experts if experts else W.NVFP4Weight
    return kind(q, s.view(torch.float8_e4m3fn), t2, orig_dtype=dtype, is_swizzled_scales=swizzled), value


def quantized_values(x: torch.Tensor, fmt: str, mode="floor", second=None) -> np.ndarray:
    """What the tokens stand for after their quantisation."""
    codes, byte = R.quantize(exact(x), fmt, mode=mode, second=second)
    return R.values(codes, byte, fmt, second)


def assert_product(got: torch.Tensor, a: np.ndarray, b: np.ndarray) -> None:
    """got = a @ b.T within the module's bound."""
    want, size = a @ b.T, np.abs(a) @ np.abs(b).T
    bound = size * a.shape[1] * 2.0 ** -23
    if got.dtype is torch.bfloat16:
        bound = bound * (1 + 2.0 ** -8) + np.abs(want) * 2.0 ** -8
    off = np.abs(exact(got) - want)
    assert np.isfinite(exact(got)).all()
    assert (off <= bound + 1e-30).all(), f"off by up to {np.max(off / (bound + 1e-30)):.3g} bounds"


# ---------------------------------------------------------------- quantisation
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("swizzled", [False, True], ids=["rows", "swizzled"])
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (70, 224), (129, 128), (64, 1056), (257, 320)])
@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_codes_and_scales(fmt, rows, cols, swizzled, dtype, cuda_device):
    x = to_torch(rng(rows, cols).standard_normal((rows, cols)) * 0.7, dtype, cuda_device)
    x[0] = 0.0
    if fmt == "mxfp4":
        w = fp4.quantize_mxfp4(x, swizzled=swizzled)
    else:
        w = fp4.quantize_nvfp4(x, two_level=False, swizzled=swizzled)
    codes, byte = R.quantize(exact(x), fmt)
    np.testing.assert_array_equal(codes_of(w), codes)
    np.testing.assert_array_equal(bytes_of(w), R.lay_out(byte, swizzled))  # padding included: zeros


@pytest.mark.parametrize("cols", [16, 48, 80, 144, 1072])
def test_nvfp4_columns_of_sixteen(cols, cuda_device):
    x = to_torch(rng(cols).standard_normal((37, cols)), torch.bfloat16, cuda_device)
    codes, byte = R.quantize(exact(x), "nvfp4")
    for swizzled in (False, True):
        w = fp4.quantize_nvfp4(x, two_level=False, swizzled=swizzled)
        np.testing.assert_array_equal(codes_of(w), codes)
        np.testing.assert_array_equal(bytes_of(w), R.lay_out(byte, swizzled))


@pytest.mark.parametrize("mode", MODES)
def test_mx_modes_over_the_whole_exponent_range(mode, cuda_device):
    g = rng(7)
    # block maxima on and around every power of two and 1.5, 1.75 and 6 times one
    tops = np.concatenate([np.float32(m) * np.float32(2.0) ** np.arange(-126, 126, dtype=np.float32)
                           for m in (1.0, 1.0 + 2 ** -23, 1.5, 1.75, 1.75 - 2 ** -23, 2 - 2 ** -23)])
    tops = np.concatenate([tops, [0.0, 1e-40, 2.0 ** -149, 3.4e38]]).astype(np.float32)
    x = (g.uniform(-1, 1, (tops.size, 32)).astype(np.float32) * tops[:, None]).astype(np.float32)
    x[np.arange(tops.size), g.integers(0, 32, tops.size)] = tops
    w = fp4.quantize_mxfp4(to_torch(x, torch.float32, cuda_device), scaling_mode=mode)
    codes, byte = R.quantize(x.astype(np.float64), "mxfp4", mode=mode)
    np.testing.assert_array_equal(bytes_of(w), byte)
    np.testing.assert_array_equal(codes_of(w), codes)


def test_rounding_ties_go_to_even(cuda_device):
    """Values exactly between two codes, for every e4m3 unit of a block."""
    units = R.E4M3[8:127]
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, -6.0])
    x = units[:, None] * ties[None, :]
    t = to_torch(x, torch.float32, cuda_device)
    assert (exact(t) == x).all()
    w = fp4.quantize_nvfp4(t, two_level=False)
    np.testing.assert_array_equal(codes_of(w), np.tile(R.encode_e2m1(ties), (units.size, 1)))
    # one unit in the last place to either side of each tie
    for toward in (0.0, np.inf):
        y = np.nextafter(x.astype(np.float32), np.float32(toward) * np.sign(x).astype(np.float32))
        y[:, 7] = x[:, 7]
        w = fp4.quantize_nvfp4(to_torch(y, torch.float32, cuda_device), two_level=False)
        codes, byte = R.quantize(y.astype(np.float64), "nvfp4")
        np.testing.assert_array_equal(bytes_of(w), byte)
        np.testing.assert_array_equal(codes_of(w), codes)


@pytest.mark.parametrize("swizzled", [False, True], ids=["rows", "swizzled"])
@pytest.mark.parametrize("shape", [(5, 64), (200, 336), (3, 40, 80), (2, 128, 256)])
def test_two_level(shape, swizzled, cuda_device):
    x = to_torch(rng(*shape).standard_normal(shape) * 0.02, torch.bfloat16, cuda_device)
    w = fp4.quantize_nvfp4(x, swizzled=swizzled)
    stack = exact(x).reshape(-1, *shape[-2:])
    second = w.per_tensor_scale.cpu().numpy()
    assert second.shape == (stack.shape[0],)
    back = exact(fp4.dequantize_fp4(w, torch.float32)).reshape(stack.shape)
    for i, m in enumerate(stack):
        assert second[i] == R.second_of(m)
        got = w if x.ndim == 2 else w.expert(i)
        codes, byte = R.quantize(m, "nvfp4", second=float(second[i]))
        np.testing.assert_array_equal(codes_of(got), codes)
        np.testing.assert_array_equal(bytes_of(got), R.lay_out(byte, swizzled))
        np.testing.assert_allclose(back[i], R.values(codes, byte, "nvfp4", float(second[i])), rtol=2.0 ** -23)
    given = fp4.quantize_nvfp4(x, per_tensor_scale=w.per_tensor_scale, swizzled=swizzled)
    assert torch.equal(given.qdata, w.qdata) and torch.equal(given.scale.view(torch.uint8), w.scale.view(torch.uint8))


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("swizzled", [False, True], ids=["rows", "swizzled"])
@pytest.mark.parametrize("shape", [(3, 700, 2080), (5, 1030, 544), (1, 9000, 96), (40, 70, 544)])
@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_many_rows_of_several_matrices(fmt, shape, swizzled, dtype, cuda_device):
    """Enough rows that a block quantises several places, with its last one in any matrix, row and column."""
    dense = rng(*shape).standard_normal(shape) * np.linspace(0.01, 1.0, shape[0])[:, None, None]
    x = to_torch(dense, dtype, cuda_device)
    w = fp4.quantize_mxfp4(x, swizzled=swizzled) if fmt == "mxfp4" else fp4.quantize_nvfp4(x, swizzled=swizzled)
    for i, m in enumerate(exact(x)):
        second = None if fmt == "mxfp4" else float(w.per_tensor_scale[i])
        assert second is None or second == R.second_of(m)
        codes, byte = R.quantize(m, fmt, second=second)
        np.testing.assert_array_equal(codes_of(w.expert(i)), codes)
        np.testing.assert_array_equal(bytes_of(w.expert(i)), R.lay_out(byte, swizzled))


def test_quantize_strided_and_unaligned_rows(cuda_device):
    base = to_torch(rng(3).standard_normal((40, 300)), torch.bfloat16, cuda_device)
    for view in (base[:, :256], base[:, 3:259], base[1::3, 8:264], base.t()[:, :32], base[::2, 5:101].t()[:64, :16]):
        for dtype in DTYPES:
            x = view.to(dtype) if dtype is not view.dtype else view
            if x.shape[1] % 32 == 0:
                w, d = fp4.quantize_mxfp4(x), fp4.quantize_mxfp4(x.contiguous())
                assert torch.equal(w.qdata, d.qdata) and torch.equal(w.scale, d.scale)
            w, d = fp4.quantize_nvfp4(x), fp4.quantize_nvfp4(x.contiguous())
            assert torch.equal(w.qdata, d.qdata) and torch.equal(w.per_tensor_scale, d.per_tensor_scale)


def test_a_single_row_may_have_any_stride(cuda_device):
    column = to_torch(rng(15).standard_normal((64, 1)), torch.bfloat16, cuda_device)
    scale = torch.tensor([0.01], device=cuda_device)
    for x in (column.t(), column.t()[:, :48]):
        assert x.stride(0) < x.shape[1]
        w = fp4.quantize_nvfp4(x, per_tensor_scale=scale)
        again = fp4.quantize_nvfp4(x.reshape(-1).clone()[None], per_tensor_scale=scale)
        assert torch.equal(w.qdata, again.qdata) and w.qdata.shape == (1, x.shape[1] // 2)
        y = fp4.linear_fp4(x, w)
        assert torch.equal(y, fp4.linear_fp4(x.reshape(-1).clone(), w)[None])
        assert torch.equal(fp4.linear_fp4_grad_input(y, w), fp4.linear_fp4_grad_input(y.reshape(-1).clone(), w)[None])


@pytest.mark.parametrize("fmt", FORMATS)
def test_nan_blocks_and_infinities(fmt, cuda_device):
    x = torch.ones((4, 128), device=cuda_device)
    x[1, 40] = float("nan")
    x[2, 50] = float("-inf")
    w = fp4.quantize_mxfp4(x) if fmt == "mxfp4" else fp4.quantize_nvfp4(x, two_level=False)
    codes, byte = R.quantize(exact(x), fmt)
    np.testing.assert_array_equal(bytes_of(w), byte)
    back = exact(fp4.dequantize_fp4(w))
    want = R.values(codes, byte, fmt)
    block = R.BLOCK[fmt]
    nan = np.zeros((4, 128), bool)
    nan[1, 40 // block * block:(40 // block + 1) * block] = True
    np.testing.assert_array_equal(np.isnan(back), nan)
    np.testing.assert_array_equal(back[~nan], np.float32(want)[~nan])
    # an infinity takes its block's largest value, which MXFP4 stores as a number beyond fp32
    assert back[2, 50] == (-np.inf if fmt == "mxfp4" else -6 * 448)


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("swizzled", [False, True], ids=["rows", "swizzled"])
@pytest.mark.parametrize("fmt", FORMATS)
def test_dequantize(fmt, swizzled, dtype, cuda_device):
    w, v = make_weight(fmt, 131, 224, cuda_device, swizzled=swizzled, second=0.37 if fmt == "nvfp4" else None, experts=3)
    got = fp4.dequantize_fp4(w, dtype)
    assert got.dtype is dtype and tuple(got.shape) == w.shape
    np.testing.assert_allclose(exact(got), v, rtol=2.0 ** -8 if dtype is torch.bfloat16 else 2.0 ** -23)


def test_quantize_then_merge_of_nothing_keeps_the_weight(cuda_device):
    """A merge with zero factors re-encodes what the quantiser made and changes nothing."""
    from piper_offload_b200 import adapters as AD

    x = to_torch(rng(11).standard_normal((256, 512)) * 0.02, torch.bfloat16, cuda_device)
    for swizzled in (False, True):
        w = fp4.quantize_mxfp4(x, swizzled=swizzled)
        before = w.qdata.clone(), w.scale.clone(), exact(fp4.dequantize_fp4(w))
        b = torch.zeros((256, 16), dtype=torch.bfloat16, device=cuda_device)
        a = torch.ones((16, 512), dtype=torch.bfloat16, device=cuda_device)
        AD.MxAdapter.merge_lora_(w, b, a, 1.0)
        np.testing.assert_array_equal(exact(fp4.dequantize_fp4(w)), before[2])


# -------------------------------------------------------------------- products
SHAPES = [(1, 128, 64), (1, 7, 32), (5, 300, 96), (16, 128, 256), (31, 129, 512), (33, 130, 544), (64, 256, 2080),
          (128, 384, 1024), (129, 250, 320), (300, 200, 800), (515, 128, 64), (700, 520, 416)]


@pytest.mark.parametrize("swizzled", [False, True], ids=["rows", "swizzled"])
@pytest.mark.parametrize("tokens,rows,cols", SHAPES)
@pytest.mark.parametrize("fmt", FORMATS)
def test_linear(fmt, tokens, rows, cols, swizzled, cuda_device):
    w, v = make_weight(fmt, rows, cols, cuda_device, swizzled=swizzled)
    x = to_torch(rng(tokens, cols).standard_normal((tokens, cols)), torch.bfloat16, cuda_device)
    assert_product(fp4.linear_fp4(x, w), quantized_values(x, fmt), v[0])


@pytest.mark.parametrize("tokens,rows,cols", [(1, 128, 256), (40, 100, 160), (300, 200, 800)])
@pytest.mark.parametrize("fmt", FORMATS)
def test_linear_fp32_tokens(fmt, tokens, rows, cols, cuda_device):
    w, v = make_weight(fmt, rows, cols, cuda_device)
    x = to_torch(rng(tokens, cols).standard_normal((tokens, cols)), torch.float32, cuda_device)
    y = fp4.linear_fp4(x, w)
    assert y.dtype is torch.float32
    assert_product(y, quantized_values(x, fmt), v[0])


@pytest.mark.parametrize("tokens", [1, 20, 200])
@pytest.mark.parametrize("cols", [16, 48, 80, 208, 1040])
def test_linear_nvfp4_columns_of_sixteen(cols, tokens, cuda_device):
    for swizzled in (False, True):
        w, v = make_weight("nvfp4", 140, cols, cuda_device, swizzled=swizzled)
        x = to_torch(rng(tokens, cols).standard_normal((tokens, cols)), torch.bfloat16, cuda_device)
        assert_product(fp4.linear_fp4(x, w), quantized_values(x, "nvfp4"), v[0])


@pytest.mark.parametrize("swizzled", [False, True], ids=["rows", "swizzled"])
@pytest.mark.parametrize("tokens", [1, 2, 20, 100, 130])
@pytest.mark.parametrize("fmt,rows,cols", [("mxfp4", 130, 4128), ("nvfp4", 130, 4112), ("nvfp4", 64, 8192), ("mxfp4", 300, 16384)])
def test_long_rows_are_split_over_a_cluster(fmt, rows, cols, tokens, swizzled, cuda_device):
    """Few outputs and many columns: several blocks share a tile's columns and add their sums up."""
    w, v = make_weight(fmt, rows, cols, cuda_device, swizzled=swizzled, second=0.25 if fmt == "nvfp4" else None)
    for dtype in DTYPES:
        x = to_torch(rng(tokens, cols).standard_normal((tokens, cols)), dtype, cuda_device)
        assert_product(fp4.linear_fp4(x, w), quantized_values(x, fmt), v[0])


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("tokens,rows,cols", [(1, 4100, 160), (40, 4096, 96), (200, 2111, 224)])
@pytest.mark.parametrize("fmt", FORMATS)
def test_long_gradients_are_split_over_a_cluster(fmt, tokens, rows, cols, dtype, cuda_device):
    w, v = make_weight(fmt, rows, cols, cuda_device)
    dy = to_torch(rng(tokens, rows).standard_normal((tokens, rows)), dtype, cuda_device)
    assert_product(fp4.linear_fp4_grad_input(dy, w), exact(dy), v[0].T)


@pytest.mark.parametrize("tokens,rows,cols", [(3000, 700, 288), (1600, 4000, 96)])
@pytest.mark.parametrize("fmt", FORMATS)
def test_many_tokens(fmt, tokens, rows, cols, cuda_device):
    """More tiles than SMs, in every direction."""
    w, v = make_weight(fmt, rows, cols, cuda_device)
    x = to_torch(rng(tokens, cols).standard_normal((tokens, cols)), torch.bfloat16, cuda_device)
    assert_product(fp4.linear_fp4(x, w), quantized_values(x, fmt), v[0])
    dy = to_torch(rng(tokens, rows).standard_normal((tokens, rows)), torch.bfloat16, cuda_device)
    assert_product(fp4.linear_fp4_grad_input(dy, w), exact(dy), v[0].T)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("cols", [96, 160, 224])
def test_scale_padding_may_hold_anything(fmt, cols, cuda_device):
    """Padding bytes of swizzled scales (here NaN codes) take no part."""
    w, v = make_weight(fmt, 70, cols, cuda_device, padding=255 if fmt == "mxfp4" else 127)
    x = to_torch(rng(cols).standard_normal((50, cols)), torch.bfloat16, cuda_device)
    assert_product(fp4.linear_fp4(x, w), quantized_values(x, fmt), v[0])
    dy = to_torch(rng(cols).standard_normal((50, 70)), torch.bfloat16, cuda_device)
    assert_product(fp4.linear_fp4_grad_input(dy, w), exact(dy), v[0].T)


@pytest.mark.parametrize("mode", MODES)
def test_linear_mx_modes(mode, cuda_device):
    w, v = make_weight("mxfp4", 100, 256, cuda_device)
    w.act_quant_kwargs = W.MXActQuantKwargs(W.MXScalingMode(mode))
    x = to_torch(rng(5).standard_normal((60, 256)), torch.bfloat16, cuda_device)
    assert_product(fp4.linear_fp4(x, w), quantized_values(x, "mxfp4", mode), v[0])


@pytest.mark.parametrize("tokens", [1, 48, 256])
def test_linear_second_level_scales(tokens, cuda_device):
    w, v = make_weight("nvfp4", 96, 192, cuda_device, second=0.25)
    x = to_torch(rng(6).standard_normal((tokens, 192)) * 5, torch.bfloat16, cuda_device)
    act = torch.full((1,), 0.03, device=cuda_device)
    y = fp4.linear_fp4(x, w, act_per_tensor_scale=act)
    assert_product(y, quantized_values(x, "nvfp4", second=float(act)), v[0])


@pytest.mark.parametrize("fmt", FORMATS)
def test_linear_shapes_strides_and_offsets(fmt, cuda_device):
    w, v = make_weight(fmt, 136, 128, cuda_device)
    base = to_torch(rng(8).standard_normal((6, 9, 300)), torch.bfloat16, cuda_device)
    for x in (base[..., :128], base[..., 5:133], base[:, 0, :128], base[0, 0, 1:129], base[:, ::2, 16:144],
              base.transpose(0, 1)[..., :128], base[0, :1, :128].expand(4, 128)):
        y = fp4.linear_fp4(x, w)
        assert y.shape == (*x.shape[:-1], 136)
        assert_product(y.reshape(-1, 136), quantized_values(x.reshape(-1, 128), fmt), v[0])
    assert fp4.linear_fp4(base[:0, 0, :128], w).shape == (0, 136)
    # codes and scales that start anywhere
    store = torch.zeros(w.qdata.numel() + 9, dtype=torch.uint8, device=cuda_device)
    sstore = torch.zeros(w.scale.numel() + 9, dtype=torch.uint8, device=cuda_device)
    x = base[:, 0, :128]
    dy = to_torch(rng(9).standard_normal((6, 136)), torch.bfloat16, cuda_device)
    want, dwant = fp4.linear_fp4(x, w), fp4.linear_fp4_grad_input(dy, w)
    for off in (1, 3, 8):
        q = store[off:off + w.qdata.numel()].view(w.qdata.shape).copy_(w.qdata)
        s = sstore[off:off + w.scale.numel()].view(torch.uint8).view(w.scale.shape).copy_(w.scale.view(torch.uint8))
        moved = (W.MXWeight(q, s, torch.float4_e2m1fn_x2, is_swizzled_scales=True) if fmt == "mxfp4" else
                 W.NVFP4Weight(q, s.view(torch.float8_e4m3fn), is_swizzled_scales=True))
        assert torch.equal(fp4.linear_fp4(x, moved), want)
        assert torch.equal(fp4.linear_fp4_grad_input(dy, moved), dwant)


def test_nan_tokens_reach_only_their_rows(cuda_device):
    for fmt in FORMATS:
        w, _ = make_weight(fmt, 160, 256, cuda_device)
        x = to_torch(rng(10).standard_normal((70, 256)), torch.bfloat16, cuda_device)
        clean = fp4.linear_fp4(x, w)
        x[3, 200] = float("nan")
        y = fp4.linear_fp4(x, w)
        assert y[3].isnan().all()
        keep = torch.arange(70, device=cuda_device) != 3
        assert torch.equal(y[keep], clean[keep])


# --------------------------------------------------------------------- experts
GROUPS = [[5], [0, 3, 0], [1, 1, 1, 1, 1, 1, 1], [130, 0, 7, 64], [33, 257, 1, 0, 0, 90], [0, 0, 0], [300, 300],
          [2] * 40, [60, 0, 2, 1, 1, 95, 0, 33], [100] + [0] * 9, [40] + [0] * 30]


@pytest.mark.parametrize("tail", [0, 37])
@pytest.mark.parametrize("swizzled", [False, True], ids=["rows", "swizzled"])
@pytest.mark.parametrize("sizes", GROUPS, ids=lambda s: "-".join(map(str, s[:8])))
@pytest.mark.parametrize("fmt", FORMATS)
def test_grouped(fmt, sizes, swizzled, tail, cuda_device):
    rows, cols = (136, 160) if fmt == "mxfp4" else (130, 208)
    tokens = sum(sizes) + tail
    w, v = make_weight(fmt, rows, cols, cuda_device, swizzled=swizzled, experts=len(sizes),
                       second=0.5 if fmt == "nvfp4" else None)
    x = to_torch(rng(tokens).standard_normal((tokens, cols)), torch.bfloat16, cuda_device)
    dy = to_torch(rng(tokens, 1).standard_normal((tokens, rows)), torch.bfloat16, cuda_device)
    ends = torch.tensor(sizes, device=cuda_device).cumsum(0).to(torch.int32)
    y, dx = fp4.grouped_linear_fp4(x, w, ends), fp4.grouped_linear_fp4_grad_input(dy, w, ends)
    xv, at = quantized_values(x, fmt), 0
    for e, n in enumerate(sizes):
        if n:
            assert_product(y[at:at + n], xv[at:at + n], v[e])
            assert_product(dx[at:at + n], exact(dy[at:at + n]), v[e].T)
        at += n
    assert not y[at:].any() and not dx[at:].any()


def test_grouped_equals_each_expert_alone(cuda_device):
    sizes = [70, 0, 200, 1]
    w, _ = make_weight("nvfp4", 256, 512, cuda_device, experts=4, second=0.5)
    x = to_torch(rng(1).standard_normal((271, 512)), torch.bfloat16, cuda_device)
    ends = torch.tensor(sizes, device=cuda_device).cumsum(0).to(torch.int32)
    y, at = fp4.grouped_linear_fp4(x, w, ends), 0
    for e, n in enumerate(sizes):
        if n:
            alone = fp4.linear_fp4(x[at:at + n], w.expert(e))
            # the two may add their sums in another order before the one rounding
            torch.testing.assert_close(y[at:at + n].float(), alone.float(), rtol=2.0 ** -7, atol=1e-4)
        at += n


def test_a_merge_into_an_expert_changes_the_stack(cuda_device):
    from piper_offload_b200 import adapters as AD

    dense = to_torch(rng(2).standard_normal((3, 128, 256)) * 0.02, torch.bfloat16, cuda_device)
    stack = fp4.quantize_nvfp4(dense)
    before = fp4.dequantize_fp4(stack)
    b = to_torch(rng(3).standard_normal((128, 8)) * 0.05, torch.bfloat16, cuda_device)
    a = to_torch(rng(4).standard_normal((8, 256)) * 0.05, torch.bfloat16, cuda_device)
    AD.Nvfp4Adapter.merge_lora_(stack.expert(1), b, a, 1.0)
    after = fp4.dequantize_fp4(stack)
    assert torch.equal(after[0], before[0]) and torch.equal(after[2], before[2])
    moved = exact(after[1]) - exact(before[1])
    want = exact(b) @ exact(a)
    assert np.linalg.norm(moved - want) < 0.35 * np.linalg.norm(want)


# ------------------------------------------------------------------- gradients
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp32"])
@pytest.mark.parametrize("swizzled", [False, True], ids=["rows", "swizzled"])
@pytest.mark.parametrize("tokens,rows,cols", [(1, 64, 64), (3, 7, 32), (33, 256, 512), (64, 131, 96), (129, 200, 416),
                                              (300, 520, 288), (520, 72, 128)])
@pytest.mark.parametrize("fmt", FORMATS)
def test_grad_input(fmt, tokens, rows, cols, swizzled, dtype, cuda_device):
    w, v = make_weight(fmt, rows, cols, cuda_device, swizzled=swizzled, second=0.3 if fmt == "nvfp4" else None)
    dy = to_torch(rng(tokens, rows).standard_normal((tokens, rows)), dtype, cuda_device)
    dx = fp4.linear_fp4_grad_input(dy, w)
    assert dx.dtype is dtype
    # the second level multiplies the fp32 sum: one more rounding, inside the bound's slack of rows * 2**-23
    assert_product(dx, exact(dy), v[0].T)


@pytest.mark.parametrize("cols", [16, 48, 80, 208])
def test_grad_input_columns_of_sixteen(cols, cuda_device):
    for swizzled in (False, True):
        w, v = make_weight("nvfp4", 140, cols, cuda_device, swizzled=swizzled)
        dy = to_torch(rng(cols).standard_normal((45, 140)), torch.bfloat16, cuda_device)
        assert_product(fp4.linear_fp4_grad_input(dy, w), exact(dy), v[0].T)


def test_grad_input_strides(cuda_device):
    w, v = make_weight("mxfp4", 128, 96, cuda_device)
    base = to_torch(rng(8).standard_normal((20, 7, 150)), torch.bfloat16, cuda_device)
    for dy in (base[..., :128], base[..., 3:131], base[0, 0, 8:136], base[::2, 1, 16:144], base[0, :1, :128].expand(5, 128)):
        dx = fp4.linear_fp4_grad_input(dy, w)
        assert dx.shape == (*dy.shape[:-1], 96)
        assert_product(dx.reshape(-1, 96), exact(dy.reshape(-1, 128)), v[0].T)
    assert fp4.linear_fp4_grad_input(base[:0, 0, :128], w).shape == (0, 96)


@pytest.mark.parametrize("fmt", FORMATS)
def test_gradients_at_the_end_of_the_range(fmt, cuda_device):
    """fp32 gradients that bf16 cannot hold, an infinity and a NaN: each reaches its own row as the formula says."""
    dense = to_torch(rng(13).standard_normal((96, 160)) * 0.02, torch.bfloat16, cuda_device)
    # no second level: it multiplies the sum, which has to stay finite before that
    w = fp4.quantize_mxfp4(dense) if fmt == "mxfp4" else fp4.quantize_nvfp4(dense, two_level=False)
    v = exact(fp4.dequantize_fp4(w, torch.float32))
    assert np.abs(v).max() < 1  # no product of a finite row overflows
    dy = to_torch(rng(14).standard_normal((40, 96)), torch.float32, cuda_device)
    dy[:4] = 0
    dy[0, 2], dy[1, 3] = torch.finfo(torch.float32).max, -3.4e38
    dy[2, 5], dy[3, 7] = float("inf"), float("nan")
    dx = fp4.linear_fp4_grad_input(dy, w)
    rows = [0, 1, *range(4, 40)]
    assert_product(dx[rows], exact(dy[rows]), v.T)
    with np.errstate(invalid="ignore"):
        np.testing.assert_array_equal(exact(dx[2]), np.inf * v[5])  # an infinity times a zero is a NaN
    assert dx[3].isnan().all()


def test_gradient_against_differences(cuda_device):
    """Along directions in which the quantised tokens move exactly (whole codes), the product is linear: its
    difference is the gradient's inner product."""
    w, _ = make_weight("nvfp4", 96, 128, cuda_device, second=0.5)
    g = rng(21)
    x = R.GRID[g.integers(0, 7, (40, 128))]
    x[:, ::16] = 6.0  # keeps every block's scale at 1
    move = np.zeros_like(x)
    at = (slice(None), slice(1, None, 16))
    move[at] = g.choice([-1.0, 1.0], x[at].shape)
    x[at] = 2.0  # 1, 2 and 3 are all codes
    t = to_torch(x, torch.float32, cuda_device).requires_grad_()
    y = fp4.linear_fp4(t, w)
    c = to_torch(g.standard_normal((40, 96)), torch.float32, cuda_device)
    y.backward(c)
    plus, minus = (fp4.linear_fp4(to_torch(x + s * move, torch.float32, cuda_device), w) for s in (1, -1))
    for row in range(40):
        want = float(((plus[row] - minus[row]).double() / 2 * c[row].double()).sum())
        got = float((t.grad[row].double().cpu() * torch.from_numpy(move[row])).sum())
        size = float(np.abs(exact(t.grad[row]) * move[row]).sum()) + abs(want)
        assert abs(got - want) <= 1e-5 * size + 1e-6


@pytest.mark.parametrize("grouped", [False, True])
def test_autograd(grouped, cuda_device):
    w, v = make_weight("mxfp4", 136, 160, cuda_device, experts=3 if grouped else None)
    x = to_torch(rng(31).standard_normal((90, 160)), torch.bfloat16, cuda_device).requires_grad_()
    dy = to_torch(rng(32).standard_normal((90, 136)), torch.bfloat16, cuda_device)
    if grouped:
        ends = torch.tensor([20, 20, 80], dtype=torch.int32, device=cuda_device)
        fp4.grouped_linear_fp4(x, w, ends).backward(dy)
        assert torch.equal(x.grad, fp4.grouped_linear_fp4_grad_input(dy, w, ends))
    else:
        fp4.linear_fp4(x, w).backward(dy)
        assert torch.equal(x.grad, fp4.linear_fp4_grad_input(dy, w))
        # broadcast gradients and a sum over several uses
        x.grad = None
        (fp4.linear_fp4(x, w).sum() + fp4.linear_fp4(x, w).sum()).backward()
        assert_product(x.grad / 2, np.ones((90, 136)), v[0].T)
    with torch.no_grad():
        assert not (fp4.grouped_linear_fp4(x, w, ends) if grouped else fp4.linear_fp4(x, w)).requires_grad


def test_changed_ends_are_noticed_before_the_backward_pass(cuda_device):
    w, _ = make_weight("mxfp4", 128, 64, cuda_device, experts=2)
    x = torch.ones((8, 64), dtype=torch.bfloat16, device=cuda_device, requires_grad=True)
    ends = torch.tensor([4, 8], dtype=torch.int32, device=cuda_device)
    y = fp4.grouped_linear_fp4(x, w, ends)
    ends[0] = 2
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


# ------------------------------------------------------- streams, graphs, repeats
def test_other_streams_and_graphs(cuda_device):
    w, _ = make_weight("nvfp4", 256, 512, cuda_device, experts=4, second=0.5)
    x = to_torch(rng(41).standard_normal((100, 512)), torch.bfloat16, cuda_device)
    ends = torch.tensor([10, 40, 40, 100], dtype=torch.int32, device=cuda_device)
    want = fp4.grouped_linear_fp4(x, w, ends)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        y = fp4.grouped_linear_fp4(x, w, ends)
    torch.cuda.current_stream().wait_stream(other)
    assert torch.equal(y, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fp4.grouped_linear_fp4(x, w, ends)
    ends.copy_(torch.tensor([0, 90, 95, 98], dtype=torch.int32))
    graph.replay()
    assert torch.equal(y, fp4.grouped_linear_fp4(x, w, ends))


@pytest.mark.parametrize("tokens", [1, 24, 300])
def test_repeats_are_bitwise_equal(tokens, cuda_device):
    w, _ = make_weight("nvfp4", 512, 2048, cuda_device)
    x = to_torch(rng(51).standard_normal((tokens, 2048)), torch.bfloat16, cuda_device)
    dy = to_torch(rng(52).standard_normal((tokens, 512)), torch.bfloat16, cuda_device)
    y, dx = fp4.linear_fp4(x, w), fp4.linear_fp4_grad_input(dy, w)
    for _ in range(5):
        assert torch.equal(fp4.linear_fp4(x, w), y) and torch.equal(fp4.linear_fp4_grad_input(dy, w), dx)


@pytest.mark.parametrize("fmt", FORMATS)
def test_compiled_calls_and_the_written_out_path_agree(fmt, cuda_device, monkeypatch):
    w, _ = make_weight(fmt, 136, 192, cuda_device, second=0.5 if fmt == "nvfp4" else None)
    stack, _ = make_weight(fmt, 136, 192, cuda_device, swizzled=False, experts=3)
    x = to_torch(rng(61).standard_normal((50, 192)), torch.bfloat16, cuda_device)
    dy = to_torch(rng(62).standard_normal((50, 136)), torch.float32, cuda_device)
    ends = torch.tensor([20, 20, 45], dtype=torch.int32, device=cuda_device)

    def results():
        packed = [fp4.quantize_mxfp4(x, scaling_mode="even", swizzled=1)] if fmt == "mxfp4" else [
            fp4.quantize_nvfp4(x), fp4.quantize_nvfp4(x.repeat(8, 8)), fp4.quantize_nvfp4(x, two_level=False, swizzled=True)]
        out = [t for p in packed for t in (p.qdata, p.scale.view(torch.uint8), fp4.dequantize_fp4(p, torch.float32))]
        out += [p.per_tensor_scale for p in packed if fmt == "nvfp4" and p.per_tensor_scale is not None]
        return out + [fp4.dequantize_fp4(stack), fp4.linear_fp4(x, w), fp4.linear_fp4(x[:3].float(), w),
                      fp4.grouped_linear_fp4(x, stack, ends), fp4.linear_fp4_grad_input(dy, w),
                      fp4.grouped_linear_fp4_grad_input(dy.bfloat16(), stack, ends)]

    class Declines:
        def __getattr__(self, name):
            return lambda *args: None

    fast = results()
    monkeypatch.setattr(nat, "calls", lambda: Declines())
    slow = results()
    assert len(fast) == len(slow)
    for a, b in zip(fast, slow):
        assert a.dtype is b.dtype and torch.equal(a, b)


def test_offsets_beyond_32_bits(cuda_device):
    """Codes, inputs and outputs whose ends lie past 2**32 bytes and 2**31 values.

    Scales are one and inputs small integers, so every sum is a multiple of 1/2 far below 2**23: exact in any order.
    """
    if torch.cuda.mem_get_info(cuda_device)[0] < 48 << 30:
        pytest.skip("needs 48 GB of device memory")
    g = torch.Generator(cuda_device).manual_seed(16)

    def codes_like(rows, cols):
        return torch.randint(0, 256, (rows, cols // 2), dtype=torch.uint8, device=cuda_device, generator=g)

    def weight(codes):
        scale = torch.full((codes.shape[0], codes.shape[1] // 16), 127, dtype=torch.uint8, device=cuda_device)
        return W.MXWeight(codes.contiguous(), scale, torch.float4_e2m1fn_x2, orig_dtype=torch.bfloat16)

    def values(codes):
        return exact(fp4.dequantize_fp4(weight(codes)))

    def integers(rows, cols, most):
        return torch.randint(-most, most + 1, (rows, cols), dtype=torch.int8, device=cuda_device, generator=g).to(torch.bfloat16)

    def tokens(rows, cols):
        x = integers(rows, cols, 4)
        x[:, ::32] = 4  # so that every block's scale is one
        return x

    # a weight of 4.6 GB of codes: its last rows in the product, its last columns in the gradient
    codes = codes_like(70000, 131072)
    w = weight(codes)
    x = tokens(2, 131072)
    y = fp4.linear_fp4(x.float(), w)
    np.testing.assert_array_equal(exact(y[:, -5:]), exact(x) @ values(codes[-5:]).T)
    dy = integers(2, 70000, 3)
    dx = fp4.linear_fp4_grad_input(dy.float(), w)
    np.testing.assert_array_equal(exact(dx[:, -32:]), exact(dy) @ values(codes[:, -16:]))
    del w
    # 2.8e9 outputs, as many gradients, and as many values to quantise
    codes = codes_like(40000, 64)
    w, v = weight(codes), values(codes)
    x = tokens(70000, 64)
    y = fp4.linear_fp4(x, w)
    assert torch.equal(y[-3:].cpu(), torch.from_numpy(exact(x[-3:]) @ v.T).to(torch.bfloat16))
    q, tail = fp4.quantize_mxfp4(y), fp4.quantize_mxfp4(y[-3:])
    assert torch.equal(q.qdata[-3:], tail.qdata) and torch.equal(q.scale[-3:], tail.scale)
    assert torch.equal(fp4.dequantize_fp4(q)[-3:], fp4.dequantize_fp4(tail))
    del q, y
    dy = integers(70000, 40000, 3)
    dx = fp4.linear_fp4_grad_input(dy, w)
    assert torch.equal(dx[-3:].cpu(), torch.from_numpy(exact(dy[-3:]) @ v).to(torch.bfloat16))


def test_launches_are_counted(cuda_device):
    w, _ = make_weight("mxfp4", 128, 128, cuda_device)
    x = torch.ones((4, 128), dtype=torch.bfloat16, device=cuda_device)
    before = nat.launches()
    fp4.linear_fp4(x, w)
    assert nat.launches() > before


# -------------------------------------------------------------------- refusals
def test_refusals(cuda_device):
    def ones(*shape, dtype=torch.bfloat16):
        return torch.ones(shape, dtype=dtype, device=cuda_device)

    for bad, match in ((ones(4, 40), "divisible by 32"), (ones(4, 64, dtype=torch.float16), "bfloat16 and float32"),
                       (ones(64), "matrix"), (ones(0, 64), "non-empty"), (ones(4, 64).cpu(), "CUDA")):
        with pytest.raises(ValueError, match=match):
            fp4.quantize_mxfp4(bad)
    with pytest.raises(ValueError, match="divisible by 16"):
        fp4.quantize_nvfp4(ones(4, 40))
    with pytest.raises(ValueError, match="scaling mode"):
        fp4.quantize_mxfp4(ones(4, 64), scaling_mode="nearest")
    with pytest.raises(ValueError, match="one float32 value per matrix"):
        fp4.quantize_nvfp4(ones(2, 4, 64), per_tensor_scale=ones(1, dtype=torch.float32))
    with pytest.raises(ValueError, match="without a second level"):
        fp4.quantize_nvfp4(ones(4, 64), two_level=False, per_tensor_scale=ones(1, dtype=torch.float32))

    mx, _ = make_weight("mxfp4", 64, 96, cuda_device)
    nv, _ = make_weight("nvfp4", 64, 96, cuda_device)
    stack, _ = make_weight("nvfp4", 64, 96, cuda_device, experts=3)
    ends = torch.tensor([1, 2, 4], dtype=torch.int32, device=cuda_device)
    for x, match in ((ones(4, 64), "columns"), (ones(4, 96, dtype=torch.float16), "bfloat16 and float32"),
                     (ones(4, 96).cpu(), "one CUDA device"), (ones(1).reshape(()), "columns")):
        with pytest.raises(ValueError, match=match):
            fp4.linear_fp4(x, nv)
    with pytest.raises(ValueError, match="64 rows|rows"):
        fp4.linear_fp4_grad_input(ones(4, 96), nv)
    with pytest.raises(ValueError, match="no second-level scale"):
        fp4.linear_fp4(ones(4, 96), mx, act_per_tensor_scale=ones(1, dtype=torch.float32))
    for act in (ones(2, dtype=torch.float32), ones(1), ones(1, dtype=torch.float32).cpu()):
        with pytest.raises(ValueError, match="one float32 value"):
            fp4.linear_fp4(ones(4, 96), nv, act_per_tensor_scale=act)
    for call in (fp4.linear_fp4, fp4.linear_fp4_grad_input):
        with pytest.raises(ValueError, match="one weight"):
            call(ones(4, 96), stack)
    for call, x in ((fp4.grouped_linear_fp4, ones(4, 96)), (fp4.grouped_linear_fp4_grad_input, ones(4, 64))):
        with pytest.raises(ValueError, match="stack of experts"):
            call(x, nv, ends)
        with pytest.raises(ValueError, match="stack of experts"):
            call(x[None], stack, ends)
        for wrong in (ends.long(), ends[:2], ends[None], torch.stack([ends, ends], 1)[:, 0]):
            with pytest.raises(ValueError, match="int32 vector"):
                call(x, stack, wrong)
        with pytest.raises(ValueError, match="one CUDA device"):
            call(x, stack, ends.cpu())

    def changed(w, **kw):
        return type(w)(**{**{k: getattr(w, k) for k in w.__dataclass_fields__}, **kw})

    x = ones(4, 96)
    for w, match in ((changed(nv, scale=nv.scale[:-1]), "scale shape"), (changed(nv, scale=mx.scale), "E4M3FN"),
                     (changed(mx, scale=mx.scale.float()), "E8M0"), (changed(mx, elem_dtype=torch.float8_e4m3fn), "e2m1"),
                     (changed(nv, qdata=nv.qdata.t().contiguous().t()), "contiguous"), (changed(nv, block_size=32), "blocks of 16"),
                     (changed(mx, block_size=16), "blocks of 32"), (changed(nv, qdata=nv.qdata.to(torch.int8)), "uint8"),
                     (changed(nv, per_tensor_scale=ones(2, dtype=torch.float32)), "one contiguous float32"),
                     (changed(nv, qdata=nv.qdata.cpu()), "CUDA"), (changed(nv, scale=nv.scale.cpu()), "one CUDA device"),
                     (changed(mx, act_quant_kwargs=W.MXActQuantKwargs(W.MXScalingMode("odd"))), "FLOOR, RCEIL"),
                     (changed(nv, is_swizzled_scales=False), "scale shape"), (changed(nv, qdata=nv.qdata[:0]), "non-empty")):
        with pytest.raises(ValueError, match=match):
            fp4.linear_fp4(x, w)
    assert nat.device_status(cuda_device) == 0
