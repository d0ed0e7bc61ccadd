"""GPU: the INT8 products and gradients against their definitions in 64 bits (int8_reference, where the bounds are derived)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import int8_reference as R
from piper_offload_b200 import _native_int8 as nat
from piper_offload_b200 import int8
from piper_offload_b200 import weights as W

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = ["bf16", "fp16", "fp32"]
KINDS = ["rows", "zero", "tensor", "tensor zero", "bnb8", "quanto", "quanto scalar"]


@pytest.fixture(autouse=True)
def device_status_clean(cuda_device):
    yield
    assert nat.device_status(cuda_device) == 0, "a bounded device wait timed out"


def rng(*key: int) -> np.random.Generator:
    return np.random.default_rng(list(key))


def name(dtype) -> str:
    return str(dtype).replace("torch.", "")


def to_torch(x: np.ndarray, dtype, device) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(x)).to(device=device, dtype=dtype)


def exact(t: torch.Tensor) -> np.ndarray:
    return t.detach().double().cpu().numpy()


def at_offset(t: torch.Tensor, offset: int) -> torch.Tensor:
    """A contiguous copy that starts `offset` elements into its storage."""
    room = torch.empty(t.numel() + offset, dtype=t.dtype, device=t.device)
    out = room[offset:].view(t.shape)
    out.copy_(t)
    return out


def make_weight(kind, rows, cols, device, *, seed=0, experts=None, offset=0, scale_dtype=torch.bfloat16, low=-128, high=127):
    """A weight (or stack) of random codes, its codes less zero points (E, rows, cols) and scales (E, rows) in 64 bits."""
    g = rng(seed, rows, cols)
    e = experts or 1
    codes = g.integers(low, high + 1, (e, rows, cols)).astype(np.int8)
    one = kind in ("tensor", "tensor zero", "quanto scalar")
    scale = torch.from_numpy(np.exp(g.normal(-6, 1, (e, 1 if one else rows, 1)))).to(scale_dtype if kind != "bnb8" else torch.float32)
    zero = g.integers(-128, 128, scale.shape).astype(np.int8) if "zero" in kind else None
    values = codes.astype(np.float64) - (0 if zero is None else zero.astype(np.float64))
    s64 = np.broadcast_to(scale.double().numpy() / (127 if kind == "bnb8" else 1), (e, rows, 1))[..., 0]
    q, s = torch.from_numpy(codes).to(device), scale.to(device)
    z = None if zero is None else torch.from_numpy(zero).to(device)
    if offset:
        q = at_offset(q, offset)
    if experts:
        return W.Int8Experts(q, s, (1, cols), zero_point=z), values, s64
    q = q[0]
    if kind == "bnb8":
        return W.Bnb8Weight(q, s.reshape(rows)), values[0], s64[0]
    if kind.startswith("quanto"):
        return W.QuantoWeight(q, s.reshape(()) if one else s[0], None if one else 0, W.QINT8), values[0], s64[0]
    return W.Int8Weight(q, s[0], (rows, cols) if one else (1, cols), zero_point=None if z is None else z[0]), values[0], s64[0]


def activations(tokens, cols, dtype, device, seed=1) -> torch.Tensor:
    g = rng(seed, tokens, cols)
    return to_torch(g.standard_normal((tokens, cols)) * np.where(g.random(cols) < 0.02, 20.0, 1.0), dtype, device)


def assert_within(got: torch.Tensor, want: np.ndarray, bound: np.ndarray) -> None:
    g = exact(got)
    assert g.shape == want.shape and np.isfinite(g).all()
    off = np.abs(g - want)
    assert (off <= bound).all(), f"off by up to {np.max(off / bound):.3g} bounds at {np.unravel_index(np.argmax(off / bound), off.shape)}"


def check_product(got, x, values, scale) -> None:
    want = R.product(exact(x), values, scale)
    assert got.dtype is x.dtype
    assert_within(got, want, R.product_bound(want, name(x.dtype)))


def check_gradient(got, dy, values, scale) -> None:
    want = R.gradient(exact(dy), values, scale)
    assert got.dtype is dy.dtype
    assert_within(got, want, R.gradient_bound(exact(dy), values, scale, want, name(dy.dtype)))


# ------------------------------------------------------------------- one weight
SHAPES = [(1, 1, 1), (1, 7, 16), (3, 128, 128), (17, 129, 40), (33, 70, 208), (130, 257, 333), (300, 200, 1040), (520, 130, 96)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("tokens,rows,cols", SHAPES)
def test_product(tokens, rows, cols, dtype, cuda_device):
    w, values, scale = make_weight("rows", rows, cols, cuda_device)
    x = activations(tokens, cols, dtype, cuda_device)
    check_product(int8.linear_int8(x, w), x, values, scale)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("tokens,rows,cols", SHAPES)
def test_gradient(tokens, rows, cols, dtype, cuda_device):
    w, values, scale = make_weight("rows", rows, cols, cuda_device)
    dy = to_torch(rng(5, tokens).standard_normal((tokens, rows)) * 1e-3, dtype, cuda_device)
    check_gradient(int8.linear_int8_grad_input(dy, w), dy, values, scale)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens", [2, 150])
def test_kinds_of_weights(tokens, kind, cuda_device):
    for scale_dtype in DTYPES:
        for cols in (272, 301):
            w, values, scale = make_weight(kind, 200, cols, cuda_device, scale_dtype=scale_dtype)
            x = activations(tokens, cols, torch.float16, cuda_device)
            check_product(int8.linear_int8(x, w), x, values, scale)
            dy = to_torch(rng(5).standard_normal((tokens, 200)), torch.float16, cuda_device)
            check_gradient(int8.linear_int8_grad_input(dy, w), dy, values, scale)


@pytest.mark.parametrize("tokens,rows,cols", [(1, 512, 4096), (9, 256, 8192), (64, 256, 16400), (260, 128, 2048), (40, 4096, 256), (600, 1000, 128)])
def test_long_sums_and_shared_tiles(tokens, rows, cols, cuda_device):
    """Few tiles and long sums, which blocks of a cluster share, and rows longer than registers hold."""
    w, values, scale = make_weight("zero", rows, cols, cuda_device)
    for dtype in (torch.bfloat16, torch.float32):
        x = activations(tokens, cols, dtype, cuda_device)
        check_product(int8.linear_int8(x, w), x, values, scale)
        dy = to_torch(rng(5, tokens).standard_normal((tokens, rows)), dtype, cuda_device)
        check_gradient(int8.linear_int8_grad_input(dy, w), dy, values, scale)


def test_largest_sums_do_not_wrap(cuda_device):
    """65536 columns of the largest codes and the furthest zero point: 65536 * 127 * 255 is below 2^31."""
    cols = nat.MAX_COLS
    q = torch.tensor([[-128], [127], [127]], dtype=torch.int8, device=cuda_device).expand(3, cols).contiguous()
    z = torch.tensor([[127], [-128], [0]], dtype=torch.int8, device=cuda_device)
    w = W.Int8Weight(q, torch.ones(3, 1, device=cuda_device), (1, cols), zero_point=z)
    x = torch.full((2, cols), 2.0, device=cuda_device)
    x[1] *= -1
    check_product(int8.linear_int8(x, w), x, np.stack([np.full(cols, v) for v in (-255.0, 255.0, 127.0)]), np.ones(3))
    x[0, ::2] = -2.0
    y = int8.linear_int8(x, w)
    assert (y[0] == 0).all()  # whole numbers cancel exactly


# ------------------------------------------------------------- the codes of tokens
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_codes_at_borders(dtype, cuda_device):
    """An identity weight gives back codes times the scale: every half-way value, and its neighbours, for many maxima."""
    cols = 512
    w = W.Int8Weight(torch.eye(cols, dtype=torch.int8, device=cuda_device), torch.ones(cols, 1, device=cuda_device), (1, cols))
    g = rng(3)
    tops = [127.0, 63.5, 1.0, 254.0, 3.0, 127 * 5.0, 1.9921875, 100.0, 1e-3, 129.0, 381.0] + list(g.uniform(0.5, 2, 40))
    rows = []
    for top in tops:
        a = float(torch.tensor(top).to(dtype))
        half = (np.arange(-127, 127) + 0.5) * a / 127
        near = torch.from_numpy(half).to(dtype)
        other = torch.nextafter(near.float(), torch.tensor(float("inf"))).to(dtype).double().numpy() if dtype is torch.float32 else near.double().numpy() * 1.01
        rows.append(np.concatenate([[a, -a / 2, a / 2, a / 4], near.double().numpy(), other])[:cols])
        rows[-1] = np.pad(rows[-1], (0, cols - len(rows[-1])))
    x = to_torch(np.clip(np.stack(rows), -np.array(tops)[:, None], np.array(tops)[:, None]), dtype, cuda_device)
    q, s = R.quantize(exact(x))
    y = int8.linear_int8(x.float(), w) if dtype is not torch.float32 else int8.linear_int8(x, w)
    np.testing.assert_array_equal(np.rint(exact(y) / np.where(s == 0, 1, s)), q)
    if dtype is not torch.float32:
        # in the token's own type the result rounds: each is the rounding of code times scale
        y = int8.linear_int8(x, w)
        assert (np.abs(exact(y) - q * s) <= R.product_bound(q * s, name(dtype))).all()


def test_fp32_codes_are_of_the_exact_quotient(cuda_device):
    cols = 1024
    w = W.Int8Weight(torch.eye(cols, dtype=torch.int8, device=cuda_device), torch.ones(cols, 1, device=cuda_device), (1, cols))
    g = rng(4)
    x = g.standard_normal((64, cols)).astype(np.float32)
    # quotients that round onto a half from either side
    top = np.abs(x).max(axis=1, keepdims=True)
    half = ((np.arange(cols) % 127 + 0.5)[None, :] * top.astype(np.float64) / 127).astype(np.float32)
    x[:, 1::3] = half[:, 1::3]
    x[:, 2::3] = np.nextafter(half[:, 2::3], np.float32(0))
    np.clip(x, -top, top, out=x)
    x[np.arange(64), 0] = top[:, 0]
    t = torch.from_numpy(x).to(cuda_device)
    q, s = R.quantize(x.astype(np.float64))
    np.testing.assert_array_equal(np.rint(exact(int8.linear_int8(t, w)) / s), q)


@pytest.mark.parametrize("power", [-148, -140, -126, -100, -65, -64, -63, 63, 64, 65, 120, 127])
def test_magnitudes_at_the_ends_of_fp32(power, cuda_device):
    cols = 96
    w = W.Int8Weight(torch.eye(cols, dtype=torch.int8, device=cuda_device), torch.full((cols, 1), 1.0, device=cuda_device), (1, cols))
    unit = rng(6).uniform(-1, 1, (4, cols))
    x = torch.from_numpy((unit * 1.99 * 2.0 ** power).astype(np.float32)).to(cuda_device)
    q, s = R.quantize(exact(x))
    got = exact(int8.linear_int8(x, w))
    # the smallest scales are held in few bits
    assert (np.abs(got - q * s) <= np.abs(q * s) * 5 * 2.0 ** -24 + (np.abs(q) + 1) * 2.0 ** -149).all()


@pytest.mark.parametrize("power", [-140, -126, -112, -60, 60, 100, 115])
def test_gradients_at_the_ends_of_fp32(power, cuda_device):
    """dy * scale from the smallest numbers to those whose products with codes near fp32's end."""
    w, values, scale = make_weight("rows", 40, 64, cuda_device, scale_dtype=torch.float32)
    w.scale.fill_(1.0)
    dy = torch.from_numpy((rng(7).uniform(-1, 1, (5, 40)) * 2.0 ** power).astype(np.float32)).to(cuda_device)
    want = R.gradient(exact(dy), values, np.ones(40))
    bound = R.gradient_bound(exact(dy), values, np.ones(40), want, "float32") + 2.0 ** -149
    if power <= -126:
        # values that are themselves below fp32's normal numbers keep 2^-25 of 2^-126's unit
        bound = bound + np.abs(values).sum(axis=0) * 2.0 ** (-126 - 25)
    assert_within(int8.linear_int8_grad_input(dy, w), want, bound)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_rows_that_are_not_finite(bad, dtype, cuda_device):
    for cols in (48, 2000):
        w, values, scale = make_weight("zero", 70, cols, cuda_device)
        x = activations(9, cols, dtype, cuda_device)
        clean = int8.linear_int8(x, w)
        x2 = x.clone()
        x2[3, cols - 1] = bad
        x2[5, 0] = bad
        y = int8.linear_int8(x2, w)
        assert y[[3, 5]].isnan().all()
        rest = [0, 1, 2, 4, 6, 7, 8]
        assert torch.equal(y[rest], clean[rest])
    dy = to_torch(rng(8).standard_normal((6, 70)), dtype, cuda_device)
    clean = int8.linear_int8_grad_input(dy, w)
    dy[2, 69] = bad
    dx = int8.linear_int8_grad_input(dy, w)
    assert not dx[2].isfinite().any()
    assert torch.equal(dx[[0, 1, 3, 4, 5]], clean[[0, 1, 3, 4, 5]])


def test_rows_of_zeros(cuda_device):
    w, _, _ = make_weight("zero", 70, 48, cuda_device)
    for dtype in DTYPES:
        x = torch.zeros(5, 48, dtype=dtype, device=cuda_device)
        assert torch.equal(int8.linear_int8(x, w), torch.zeros(5, 70, dtype=dtype, device=cuda_device))
        assert torch.equal(int8.linear_int8_grad_input(torch.zeros(5, 70, dtype=dtype, device=cuda_device), w), x)


# ---------------------------------------------------------------- strides and shapes
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_strides_and_alignment(dtype, cuda_device):
    base = activations(40, 700, dtype, cuda_device)
    w, values, scale = make_weight("zero", 90, 304, cuda_device)
    for x in (base[:, 3:307], base[::2, 8:312], base[1:2, 5:309], base[:, :304].t().contiguous().t(), base[:20, :304].view(4, 5, 304),
              base[0, 1:305], base[:1, :304].expand(7, 304)):
        flat = x.reshape(-1, 304)
        y = int8.linear_int8(x, w)
        assert y.shape == (*x.shape[:-1], 90)
        check_product(y.reshape(-1, 90), flat, values, scale)
    for dy in (base[:, 3:93], base[::2, 8:98], base[:, :90].t().contiguous().t(), base[0, 1:91]):
        dx = int8.linear_int8_grad_input(dy, w)
        assert dx.shape == (*dy.shape[:-1], 304)
        check_gradient(dx.reshape(-1, 304), dy.reshape(-1, 90), values, scale)


@pytest.mark.parametrize("offset", [1, 2, 7, 8, 16])
@pytest.mark.parametrize("cols", [33, 48, 130])
def test_codes_at_any_address(cols, offset, cuda_device):
    w, values, scale = make_weight("rows", 150, cols, cuda_device, offset=offset)
    x = activations(70, cols, torch.bfloat16, cuda_device)
    check_product(int8.linear_int8(x, w), x, values, scale)
    dy = to_torch(rng(5).standard_normal((70, 150)), torch.bfloat16, cuda_device)
    check_gradient(int8.linear_int8_grad_input(dy, w), dy, values, scale)


def test_no_tokens(cuda_device):
    w, _, _ = make_weight("rows", 20, 32, cuda_device)
    assert int8.linear_int8(torch.empty(0, 32, device=cuda_device), w).shape == (0, 20)
    assert int8.linear_int8_grad_input(torch.empty(2, 0, 20, device=cuda_device), w).shape == (2, 0, 32)


# ---------------------------------------------------------------------- experts
def grouped_reference(x, values, scale, ends, grad):
    out = np.zeros((x.shape[0], values.shape[2 if grad else 1]))
    bound = np.zeros_like(out)
    start = 0
    for e, end in enumerate(ends):
        end = max(start, min(max(int(end), 0), x.shape[0]))
        rows = x[start:end]
        if end > start:
            if grad:
                out[start:end] = R.gradient(exact(rows), values[e], scale[e])
                bound[start:end] = R.gradient_bound(exact(rows), values[e], scale[e], out[start:end], name(x.dtype))
            else:
                out[start:end] = R.product(exact(rows), values[e], scale[e])
                bound[start:end] = R.product_bound(out[start:end], name(x.dtype))
        start = end
    return out, bound


GROUPS = [[3, 3, 10, 40], [0, 0, 0, 40], [1, 2, 3, 4], [40, 40, 40, 40], [0, 0, 0, 0], [9, 5, 30, 20], [50, 10, 60, 3], [-4, 7, 7, 33]]


@pytest.mark.parametrize("kind", ["rows", "zero"])
@pytest.mark.parametrize("ends", GROUPS, ids=lambda e: "-".join(map(str, e)))
def test_groups(ends, kind, cuda_device):
    for dtype in DTYPES:
        w, values, scale = make_weight(kind, 137, 160, cuda_device, experts=4)
        x = activations(40, 160, dtype, cuda_device)
        e = torch.tensor(ends, dtype=torch.int32, device=cuda_device)
        y = int8.grouped_linear_int8(x, w, e)
        assert_within(y, *grouped_reference(x, values, scale, ends, False))
        dy = to_torch(rng(5).standard_normal((40, 137)), dtype, cuda_device)
        dx = int8.grouped_linear_int8_grad_input(dy, w, e)
        assert_within(dx, *grouped_reference(dy, values, scale, ends, True))


@pytest.mark.parametrize("experts,tokens,rows,cols", [(1, 300, 130, 144), (40, 900, 260, 272), (70, 64, 128, 208), (5, 1500, 300, 1031), (33, 33, 16, 16)])
def test_many_groups(experts, tokens, rows, cols, cuda_device):
    g = rng(experts, tokens)
    ends = np.sort(g.integers(0, tokens + 1, experts))
    w, values, scale = make_weight("zero", rows, cols, cuda_device, experts=experts)
    x = activations(tokens, cols, torch.bfloat16, cuda_device)
    e = torch.from_numpy(ends.astype(np.int32)).to(cuda_device)
    assert_within(int8.grouped_linear_int8(x, w, e), *grouped_reference(x, values, scale, ends, False))
    dy = to_torch(g.standard_normal((tokens, rows)), torch.bfloat16, cuda_device)
    assert_within(int8.grouped_linear_int8_grad_input(dy, w, e), *grouped_reference(dy, values, scale, ends, True))


def test_values_in_rows_of_no_expert_do_not_matter(cuda_device):
    w, values, scale = make_weight("rows", 70, 96, cuda_device, experts=3)
    x = activations(30, 96, torch.bfloat16, cuda_device)
    dy = to_torch(rng(5).standard_normal((30, 70)), torch.bfloat16, cuda_device)
    ends = torch.tensor([4, 4, 20], dtype=torch.int32, device=cuda_device)
    clean, clean_grad = int8.grouped_linear_int8(x, w, ends), int8.grouped_linear_int8_grad_input(dy, w, ends)
    x[20:], dy[20:] = float("nan"), float("inf")
    assert torch.equal(int8.grouped_linear_int8(x, w, ends), clean) and torch.equal(int8.grouped_linear_int8_grad_input(dy, w, ends), clean_grad)
    assert not clean[20:].any() and not clean_grad[20:].any()


# ------------------------------------------------------------------- derivatives
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_backward_is_the_gradient(dtype, cuda_device):
    w, values, scale = make_weight("zero", 90, 112, cuda_device)
    x = activations(20, 112, dtype, cuda_device).view(4, 5, 112).requires_grad_()
    g = to_torch(rng(5).standard_normal((4, 5, 90)), dtype, cuda_device)
    y = int8.linear_int8(x, w)
    y.backward(g)
    assert torch.equal(x.grad, int8.linear_int8_grad_input(g, w))
    check_product(y.reshape(-1, 90), x.reshape(-1, 112), values, scale)
    # a gradient that is one number for all, as a sum's is
    x.grad = None
    int8.linear_int8(x, w).sum().backward()
    check_gradient(x.grad.reshape(-1, 112), torch.ones(20, 90, dtype=dtype, device=cuda_device), values, scale)


def test_gradient_against_differences(cuda_device):
    """Codes that stay the same under the step, so the product is linear there: y(x + h) - y(x) = h * dx, with a maximum that
    does not move. h is one whole code, taken from a row whose scale is 1."""
    cols, rows = 64, 80
    w, values, scale = make_weight("rows", rows, cols, cuda_device, scale_dtype=torch.float32)
    x = torch.from_numpy(rng(2).integers(-100, 101, (3, cols)).astype(np.float32)).to(cuda_device)
    x[:, 0] = 127.0
    g = torch.from_numpy(rng(3).standard_normal((3, rows)).astype(np.float32)).to(cuda_device)
    dx = exact(int8.linear_int8_grad_input(g, w))
    for k in (1, 17, 63):
        up, down = x.clone(), x.clone()
        up[:, k] += 1
        down[:, k] -= 1
        difference = (exact(g) * (exact(int8.linear_int8(up, w)) - exact(int8.linear_int8(down, w))) / 2).sum(axis=1)
        # each product is within its bound, differences of two and halved; the gradient within its own
        far = (np.abs(exact(g)) * R.product_bound(np.abs(R.product(exact(up), values, scale)) + np.abs(R.product(exact(down), values, scale)), "float32")).sum(axis=1)
        own = R.gradient_bound(exact(g), values, scale, dx, "float32")[:, k]
        assert (np.abs(difference - dx[:, k]) <= far + own).all()


def test_grouped_backward_and_frozen_weights(cuda_device):
    w, values, scale = make_weight("rows", 90, 112, cuda_device, experts=3)
    x = activations(20, 112, torch.bfloat16, cuda_device).requires_grad_()
    ends = torch.tensor([7, 7, 18], dtype=torch.int32, device=cuda_device)
    g = to_torch(rng(5).standard_normal((20, 90)), torch.bfloat16, cuda_device)
    y = int8.grouped_linear_int8(x, w, ends)
    want = int8.grouped_linear_int8_grad_input(g, w, ends)
    held = w.scale
    w.scale = torch.zeros_like(held)  # another tensor in its place changes nothing
    y.backward(g)
    assert torch.equal(x.grad, want)
    w.scale = held
    y = int8.grouped_linear_int8(x, w, ends)
    w.scale.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(g)
    y = int8.grouped_linear_int8(x, w, ends)
    ends.add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(g)


# ------------------------------------------------------- streams, graphs, same bits
def test_same_bits_on_every_run(cuda_device):
    for tokens, rows, cols in ((5, 256, 4096), (300, 512, 1024)):
        w, _, _ = make_weight("zero", rows, cols, cuda_device)
        x = activations(tokens, cols, torch.bfloat16, cuda_device)
        dy = to_torch(rng(5).standard_normal((tokens, rows)), torch.bfloat16, cuda_device)
        first, grad = int8.linear_int8(x, w), int8.linear_int8_grad_input(dy, w)
        for _ in range(20):
            assert torch.equal(int8.linear_int8(x, w), first) and torch.equal(int8.linear_int8_grad_input(dy, w), grad)


def test_on_another_stream(cuda_device):
    w, values, scale = make_weight("rows", 500, 1024, cuda_device)
    side = torch.cuda.Stream()
    x = activations(64, 1024, torch.bfloat16, cuda_device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = int8.linear_int8(x, w)
        dx = int8.linear_int8_grad_input(y, w)
    torch.cuda.current_stream().wait_stream(side)
    check_product(y, x, values, scale)
    check_gradient(dx, y, values, scale)


def test_captured_graphs_replay(cuda_device):
    """Two graphs over the same weight, replayed in turn and on new inputs; a call before the capture makes no difference."""
    w, values, scale = make_weight("zero", 300, 544, cuda_device, experts=4)
    graphs = []
    for tokens in (33, 200):
        x = activations(tokens, 544, torch.bfloat16, cuda_device)
        ends = torch.tensor([tokens // 4, tokens // 3, tokens // 2, tokens - 5], dtype=torch.int32, device=cuda_device)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = int8.grouped_linear_int8(x, w, ends)
            dx = int8.grouped_linear_int8_grad_input(y, w, ends)
        graphs.append((graph, x, ends, y, dx))
    for turn in range(3):
        for graph, x, ends, y, dx in graphs:
            x.copy_(activations(x.shape[0], 544, torch.bfloat16, cuda_device, seed=turn))
            ends[1] = x.shape[0] // 3 + turn
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, x, ends, y, dx in graphs:
            assert_within(y, *grouped_reference(x, values, scale, ends.tolist(), False))
            assert_within(dx, *grouped_reference(y, values, scale, ends.tolist(), True))


def test_bad_arguments_are_refused(cuda_device):
    w, _, _ = make_weight("rows", 40, 64, cuda_device)
    stack, _, _ = make_weight("rows", 40, 64, cuda_device, experts=3)
    x = torch.ones(4, 64, dtype=torch.bfloat16, device=cuda_device)
    ends = torch.tensor([1, 2, 4], dtype=torch.int32, device=cuda_device)
    per_column = W.QuantoWeight(w.qdata, torch.ones(1, 64, dtype=torch.bfloat16, device=cuda_device), -1, W.QINT8)
    grouped = W.Int8Weight(w.qdata, torch.ones(40, 2, device=cuda_device), (1, 32))
    scaled = W.Int8Weight(w.qdata, w.scale, (1, 64), act_pre_scale=torch.ones(64, device=cuda_device))
    for call, match in ((lambda: int8.linear_int8(x[:, :63], w), "64 columns"), (lambda: int8.linear_int8(x.double(), w), "float64"),
                        (lambda: int8.linear_int8(x.cpu(), w), "one CUDA device"), (lambda: int8.linear_int8(x, stack), "one weight"),
                        (lambda: int8.grouped_linear_int8(x, w, ends), "stack"), (lambda: int8.grouped_linear_int8(x[None], stack, ends), "rank-two"),
                        (lambda: int8.grouped_linear_int8(x, stack, ends.long()), "int32"), (lambda: int8.grouped_linear_int8(x, stack, ends[:2]), "int32"),
                        (lambda: int8.grouped_linear_int8(x, stack, ends.cpu()), "one CUDA device"),
                        (lambda: int8.linear_int8_grad_input(x, w), "40 rows"), (lambda: int8.linear_int8(x, per_column), "columns"),
                        (lambda: int8.linear_int8(x, grouped), "for each row"), (lambda: int8.linear_int8(x, scaled), "act_pre_scale"),
                        (lambda: int8.linear_int8(x, W.Int8Weight(w.qdata, w.scale[:39], (1, 64))), "scale shape"),
                        (lambda: int8.linear_int8(x, W.Int8Weight(w.qdata, w.scale.double(), (1, 64))), "scales are"),
                        (lambda: int8.linear_int8(x, W.Int8Weight(w.qdata, w.scale, (1, 64), zero_point=w.scale)), "zero points"),
                        (lambda: int8.linear_int8(x, W.Int8Weight(w.qdata.t().contiguous().t(), w.scale, (1, 64))), "contiguous"),
                        (lambda: int8.linear_int8(torch.ones(1, nat.MAX_COLS + 16, device=cuda_device), W.Int8Weight(
                            torch.ones(1, nat.MAX_COLS + 16, dtype=torch.int8, device=cuda_device), w.scale[:1], (1, nat.MAX_COLS + 16))), "65536")):
        with pytest.raises(ValueError, match=match):
            call()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, x)
        for call in (lambda: int8.linear_int8(dual, w), lambda: int8.grouped_linear_int8(dual, stack, ends),
                     lambda: int8.linear_int8_grad_input(dual[:, :40], w)):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
