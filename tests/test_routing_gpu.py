"""GPU: expert routing and the exchange of tokens against their definitions in 64 bits (routing_reference)."""

from __future__ import annotations

import itertools

import numpy as np
import pytest
import torch

import routing_reference as R
from piper_offload_b200 import routing

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = ["bf16", "fp16", "fp32"]


def rng(*key: int) -> np.random.Generator:
    return np.random.default_rng(list(key))


def name(dtype) -> str:
    return str(dtype).replace("torch.", "")


def to_torch(x: np.ndarray, dtype, device) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(x)).to(device=device, dtype=dtype)


def exact(t: torch.Tensor) -> np.ndarray:
    return t.detach().double().cpu().numpy()


def arguments(rules: dict, device) -> dict:
    out = dict(rules)
    if out.get("bias") is not None:
        out["bias"] = torch.from_numpy(out["bias"]).to(device)
    if out.get("mask") is not None:
        out["mask"] = torch.from_numpy(out["mask"]).to(device)
    return out


def reference_rules(rules: dict) -> dict:
    out = dict(rules)
    if out.get("bias") is not None:
        out["bias"] = out["bias"].astype(np.float64)
    return out


def check_route(logits: torch.Tensor, top_k: int, **rules) -> routing.Routing:
    """All outputs against the definition; whole numbers have to be equal."""
    r = routing.route_tokens(logits, top_k, **arguments(rules, logits.device))
    l64 = exact(logits)
    weights, experts, ends, rows, source = R.route(l64, top_k, **reference_rules(rules))
    np.testing.assert_array_equal(r.experts.cpu().numpy(), experts)
    np.testing.assert_array_equal(r.ends.cpu().numpy(), ends)
    np.testing.assert_array_equal(r.rows.cpu().numpy(), rows)
    np.testing.assert_array_equal(r.source.cpu().numpy(), source)
    got = exact(r.weights)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(weights))
    for t in range(l64.shape[0]):
        ok = ~np.isnan(weights[t])
        assert (np.abs(got[t] - weights[t])[ok] <= (np.abs(weights[t]) * R.unit(l64[t]) + 2.0 ** -126)[ok]).all()
    return r


def check_gradient(logits: torch.Tensor, top_k: int, **rules) -> None:
    g = rng(9, *logits.shape).standard_normal((logits.shape[0], top_k)).astype(np.float32)
    leaf = logits.detach().clone().requires_grad_()
    r = routing.route_tokens(leaf, top_k, **arguments(rules, logits.device))
    r.weights.backward(torch.from_numpy(g).to(logits.device))
    got, l64 = exact(leaf.grad), exact(logits)
    want, size = R.gradient(l64, r.experts.cpu().numpy(), g.astype(np.float64), **reference_rules(rules))
    units = np.array([R.unit(row) for row in l64])[:, None]
    # a gradient has a weight, a difference of two sums with weights, and a quotient more than a weight has: four times its unit
    bound = 4 * units * size * (1 + HALF(logits)) + np.abs(want) * HALF(logits) + R.TINY[name(logits.dtype)] + 2.0 ** -126
    assert leaf.grad.dtype is logits.dtype and got.shape == want.shape
    assert (np.abs(got - want) <= bound).all(), f"off by up to {np.max(np.abs(got - want) / bound):.3g} bounds"


def HALF(t: torch.Tensor) -> float:
    return R.HALF_STEP[name(t.dtype)]


def normal_logits(tokens, experts, dtype, device, seed=0, std=1.5) -> torch.Tensor:
    return to_torch(rng(seed, tokens, experts).standard_normal((tokens, experts)) * std, dtype, device)


# ------------------------------------------------------------------------ choices
SHAPES = [(1, 1, 1), (1, 8, 2), (3, 5, 5), (40, 8, 2), (129, 60, 4), (200, 64, 8), (31, 33, 32), (257, 128, 1), (150, 256, 8), (20, 300, 6),
          (30, 1024, 32)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens,experts,top_k", SHAPES)
def test_route(tokens, experts, top_k, scoring, dtype, cuda_device):
    logits = normal_logits(tokens, experts, dtype, cuda_device)
    for renormalize, scale in ((True, 1.0), (False, 2.5)):
        check_route(logits, top_k, scoring=scoring, renormalize=renormalize, scale=scale)
        check_gradient(logits, top_k, scoring=scoring, renormalize=renormalize, scale=scale)


GROUPED = [(16, 4, 2, 3), (64, 8, 4, 6), (60, 5, 3, 8), (256, 8, 4, 8), (96, 32, 1, 3), (160, 2, 1, 8), (512, 16, 16, 4), (12, 12, 7, 5)]


@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("biased", [False, True], ids=["plain", "biased"])
@pytest.mark.parametrize("experts,groups,top_groups,top_k", GROUPED)
def test_groups_of_experts(experts, groups, top_groups, top_k, biased, group_score, cuda_device):
    bias = (rng(3, experts).standard_normal(experts) * 0.1).astype(np.float32) if biased else None
    for scoring, dtype in itertools.product(("softmax", "sigmoid"), (torch.bfloat16, torch.float32)):
        logits = normal_logits(150, experts, dtype, cuda_device)
        rules = {"scoring": scoring, "bias": bias, "groups": groups, "top_groups": top_groups, "group_score": group_score}
        check_route(logits, top_k, **rules)
        check_gradient(logits, top_k, **rules)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_bias_of_choices(scoring, cuda_device):
    """A bias changes who is chosen and in which order, not what a score weighs."""
    logits = normal_logits(300, 64, torch.float32, cuda_device)
    for size in (0.0, 0.01, 3.0, 1000.0):
        check_route(logits, 6, scoring=scoring, bias=(rng(4).standard_normal(64) * size).astype(np.float32))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,group_score", [(1, "max"), (8, "max"), (8, "top2")])
def test_scores_that_fp32_cannot_tell_apart(groups, group_score, scoring, cuda_device):
    """Biases that bring all choice scores within some 1e-8 of one number: the 64-bit sums decide."""
    experts = 64
    l64 = exact(normal_logits(1, experts, torch.float32, cuda_device))[0]
    bias = (0.7 - R.scores_of(l64, scoring)).astype(np.float32)
    logits = to_torch(np.tile(l64, (200, 1)), torch.float32, cuda_device)
    logits[100:] = normal_logits(100, experts, torch.float32, cuda_device, seed=5, std=1e-6) + logits[0]
    choice = R.scores_of(l64, scoring) + bias
    assert np.unique(choice.astype(np.float32)).size < 4 and np.unique(choice).size == experts
    check_route(logits, 8, scoring=scoring, bias=bias, groups=groups, top_groups=max(1, groups // 2), group_score=group_score)


def test_equal_scores_go_by_index(cuda_device):
    logits = torch.zeros(70, 96, device=cuda_device)
    for rules in ({}, {"scoring": "sigmoid"}, {"bias": np.zeros(96, np.float32)}, {"groups": 8, "top_groups": 3, "group_score": "top2"},
                  {"bias": np.full(96, 0.25, np.float32), "groups": 4, "top_groups": 2, "scoring": "sigmoid"}):
        r = check_route(logits, 5, **rules)
        assert r.experts.cpu().tolist() == [[0, 1, 2, 3, 4]] * 70
    few = to_torch(rng(2).integers(-1, 2, (200, 130)).astype(float), torch.bfloat16, cuda_device)
    for rules in ({}, {"scoring": "sigmoid"}, {"groups": 13, "top_groups": 4}):
        check_route(few, 8, **rules)
    signed = torch.tensor([[-0.0, 0.0, -0.0, -1.0]], device=cuda_device)
    assert routing.route_tokens(signed, 4).experts[0].tolist() == [0, 1, 2, 3]


def test_closed_experts(cuda_device):
    """-infinity in a logit or a bias closes an expert; tokens may run out of them."""
    g = rng(6)
    l64 = g.standard_normal((150, 24))
    l64[g.random((150, 24)) < 0.6] = -np.inf
    l64[7] = -np.inf
    l64[8, 1:] = -np.inf
    bias = np.where(g.random(24) < 0.2, -np.inf, g.standard_normal(24) * 0.1).astype(np.float32)
    for dtype, scoring, renormalize in itertools.product(DTYPES, ("softmax", "sigmoid"), (True, False)):
        logits = to_torch(l64, dtype, cuda_device)
        for rules in ({}, {"bias": bias}, {"groups": 6, "top_groups": 2, "group_score": "top2"}, {"bias": bias, "groups": 4, "top_groups": 4},
                      {"groups": 3, "top_groups": 2}):
            rules = {**rules, "scoring": scoring, "renormalize": renormalize}
            r = check_route(logits, 6, **rules)
            assert r.experts[7].eq(-1).all() and not r.weights[7].any()
            assert int(r.ends[-1]) == int((r.experts >= 0).sum())
            check_gradient(logits, 6, **rules)


def test_masked_tokens(cuda_device):
    for tokens in (20, 500):
        logits = normal_logits(tokens, 40, torch.bfloat16, cuda_device)
        for mask in (rng(7, tokens).random(tokens) < 0.7, np.zeros(tokens, bool), np.ones(tokens, bool)):
            for rules in ({}, {"scoring": "sigmoid", "renormalize": False}, {"renormalize": False}):
                r = check_route(logits, 4, mask=mask, **rules)
                assert r.experts.cpu().numpy()[~mask].max(initial=-1) == -1
                check_gradient(logits, 4, mask=mask, **rules)
        hidden = logits.clone()
        hidden[0] = float("nan")
        mask = np.arange(tokens) > 0
        r = routing.route_tokens(hidden, 4, mask=torch.from_numpy(mask).to(cuda_device))
        assert r.weights.isfinite().all() and int(r.ends[-1]) == 4 * (tokens - 1)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_logits_that_are_not_finite(value, cuda_device):
    l64 = rng(8).standard_normal((60, 40))
    l64[3, 5] = l64[4, :38] = value
    l64[5] = value
    for dtype in DTYPES:
        logits = to_torch(l64, dtype, cuda_device)
        for rules in ({}, {"renormalize": False}, {"scoring": "sigmoid"}, {"scoring": "sigmoid", "renormalize": False},
                      {"bias": np.linspace(-1, 1, 40).astype(np.float32)}, {"bias": np.linspace(-1, 1, 40).astype(np.float32), "scoring": "sigmoid"}):
            r = check_route(logits, 4, **rules)
            assert r.weights[[0, 1, 2, 6, 30]].isfinite().all()


def test_scores_too_small_for_a_number(cuda_device):
    """Choices far below the largest logit keep their shares, and sigmoids below 2^-100 theirs of that."""
    l64 = np.full((5, 16), 200.0)
    l64[:, 8:] = rng(9).standard_normal((5, 8)) - 100
    logits = to_torch(l64, torch.float32, cuda_device)
    r = check_route(logits, 3, groups=2, top_groups=1, bias=np.repeat([-1000.0, 0.0], 8).astype(np.float32))
    assert (r.experts >= 8).all()
    low = to_torch(rng(10).standard_normal((5, 16)) * 5 - 80, torch.float32, cuda_device)
    check_route(low, 3, scoring="sigmoid")
    check_gradient(low, 3, scoring="sigmoid")
    check_gradient(logits, 3, groups=2, top_groups=1, bias=np.repeat([-1000.0, 0.0], 8).astype(np.float32))


def test_strides_and_no_tokens(cuda_device):
    base = normal_logits(90, 100, torch.bfloat16, cuda_device)
    for logits in (base[:, 3:43], base[::2, :40], base.t(), base[5:6, 1:41], base[:1, :40].expand(6, 40)):
        check_route(logits, 4)
        check_gradient(logits, 4)
    r = routing.route_tokens(base[:0], 4)
    assert r.weights.shape == (0, 4) and r.source.shape == (0,) and not r.ends.any()
    leaf = base[:0].clone().requires_grad_()
    routing.route_tokens(leaf, 4).weights.sum().backward()
    assert leaf.grad.shape == (0, 100)


@pytest.mark.parametrize("tokens", [127, 128, 129, 1183, 1184, 1185, 5000, 40000])
def test_order_of_many_tokens(tokens, cuda_device):
    """The order by expert on either side of one block's tokens and in several rounds of a block's."""
    for experts, top_k in ((7, 3), (256, 8), (700, 2)):
        logits = normal_logits(tokens, experts, torch.bfloat16, cuda_device)
        mask = torch.rand(tokens, device=cuda_device, generator=torch.Generator(device=cuda_device).manual_seed(tokens)) < 0.9
        r = routing.route_tokens(logits, top_k, mask=mask)
        flat = r.experts.reshape(-1).long()
        flat = torch.where(flat < 0, experts, flat)
        order = torch.sort(flat, stable=True).indices
        count = int((flat < experts).sum())
        assert count == int(mask.sum()) * top_k
        assert torch.equal(r.source[:count].long(), order[:count]) and r.source[count:].eq(-1).all()
        assert torch.equal(r.ends.long(), torch.bincount(flat, minlength=experts + 1)[:experts].cumsum(0))
        assert torch.equal(r.rows.reshape(-1)[order[:count]].long(), torch.arange(count, device=cuda_device))
        assert r.rows.reshape(-1)[order[count:]].eq(-1).all()


# ---------------------------------------------------------------------- derivatives
def test_gradient_against_differences(cuda_device):
    for scoring, renormalize in itertools.product(("softmax", "sigmoid"), (True, False)):
        logits = normal_logits(4, 12, torch.float32, cuda_device)
        g = rng(11).standard_normal((4, 3))
        rules = {"scoring": scoring, "renormalize": renormalize, "scale": 1.5}
        leaf = logits.clone().requires_grad_()
        r = routing.route_tokens(leaf, 3, **rules)
        r.weights.backward(to_torch(g, torch.float32, cuda_device))
        l64, experts, h = exact(logits), r.experts.cpu().numpy(), 1e-4
        for t, e in itertools.product(range(4), range(12)):
            up, down = l64[t].copy(), l64[t].copy()
            up[e] += h
            down[e] -= h
            want = (g[t] * (R.weights_of(up, list(experts[t]), **rules) - R.weights_of(down, list(experts[t]), **rules))).sum() / (2 * h)
            # third derivatives of a weight are below 1, h^2 / 6 of them; fp32's share as in check_gradient
            assert abs(exact(leaf.grad)[t, e] - want) <= 1.5 * np.abs(g[t]).sum() * (h * h / 6 + 8 * R.unit(l64[t])) + 1e-9


# ------------------------------------------------------------------------ exchange
def made_routing(tokens, experts, top_k, device, masked=0.2, seed=0):
    logits = normal_logits(tokens, experts, torch.float32, device, seed=seed)
    mask = torch.from_numpy(rng(12, tokens).random(tokens) >= masked).to(device)
    return routing.route_tokens(logits, top_k, mask=mask, renormalize=False)


EXCHANGES = [(1, 3, 1, 1), (5, 4, 2, 7), (24, 8, 2, 4096), (130, 16, 8, 64), (33, 9, 9, 1030), (40, 40, 32, 96), (6000, 8, 3, 72)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("tokens,experts,top_k,hidden", EXCHANGES)
def test_exchange(tokens, experts, top_k, hidden, dtype, cuda_device):
    r = made_routing(tokens, experts, top_k, cuda_device)
    rows, source = r.rows.cpu().numpy(), r.source.cpu().numpy()
    g = rng(13, tokens, hidden)
    x = to_torch(g.standard_normal((tokens, hidden)), dtype, cuda_device).requires_grad_()
    y = to_torch(g.standard_normal((tokens * top_k, hidden)), dtype, cuda_device).requires_grad_()
    gx = to_torch(g.standard_normal((tokens * top_k, hidden)), dtype, cuda_device)
    gy = to_torch(g.standard_normal((tokens, hidden)), dtype, cuda_device)
    r.weights.requires_grad_()
    sent, back = routing.dispatch_tokens(x, r), routing.combine_tokens(y, r)
    sent.backward(gx)
    back.backward(gy)
    half, tiny = R.HALF_STEP[name(dtype)], R.TINY[name(dtype)]

    want = np.where(source[:, None] >= 0, exact(x)[np.maximum(source, 0) // top_k], 0.0)
    np.testing.assert_array_equal(exact(sent), want)

    def added(t, w):
        parts = np.where(rows[..., None] >= 0, exact(t)[np.maximum(rows, 0)], 0.0) * w[..., None]
        return parts.sum(axis=1), np.abs(parts).sum(axis=1)

    for got, t, w in ((back, y, exact(r.weights)), (x.grad, gx, np.ones(rows.shape))):
        want, size = added(t, w)
        # top_k fused additions in fp32, then the result's rounding
        assert (np.abs(exact(got) - want) <= size * top_k * 2.0 ** -24 * 1.01 + np.abs(want) * half * 1.01 + tiny).all()
    want = np.where(source[:, None] >= 0, exact(gy)[np.maximum(source, 0) // top_k] * exact(r.weights).reshape(-1, 1)[np.maximum(source, 0)], 0.0)
    assert (np.abs(exact(y.grad) - want) <= np.abs(want) * (half + 2.0 ** -24) * 1.01 + tiny).all()
    parts = np.where(rows[..., None] >= 0, exact(y)[np.maximum(rows, 0)], 0.0) * exact(gy)[:, None]
    # at most so many additions in a row for one number: a lane's, the warp's, the block's
    chain = hidden / 32 + 8 + 16
    assert (np.abs(exact(r.weights.grad) - parts.sum(-1)) <= np.abs(parts).sum(-1) * chain * 2.0 ** -24 + 2.0 ** -149).all()


def test_exchange_of_strided_rows(cuda_device):
    r = made_routing(30, 6, 2, cuda_device)
    base = normal_logits(200, 300, torch.bfloat16, cuda_device)
    for x in (base[:30, 1:129], base[:60:2, :128], base[:128, :30].t(), base[:1, :128].expand(30, 128)):
        assert torch.equal(routing.dispatch_tokens(x, r), routing.dispatch_tokens(x.contiguous(), r))
    for y in (base[:60, 1:129], base[:120:2, :128], base[:128, :60].t(), base[:1, :128].expand(60, 128)):
        assert torch.equal(routing.combine_tokens(y, r), routing.combine_tokens(y.contiguous(), r))
        one, two = y.detach().requires_grad_(), y.contiguous().requires_grad_()
        for t in (one, two):
            routing.combine_tokens(t, r).sum().backward()
        assert torch.equal(one.grad, two.grad)
    for t in (base[:30, :129], base[:30, 3:132]):
        leaf = t.detach().requires_grad_()
        routing.dispatch_tokens(leaf, r).sum().backward()
        assert torch.equal(leaf.grad.float()[:, 0], (r.rows >= 0).sum(1).float())


def test_rows_outside_count_as_none(cuda_device):
    """A routing that was not made by route_tokens: places outside the rows are neither read nor written."""
    rows = torch.tensor([[0, 900], [-5, 1], [2, 6], [3, 2 ** 31 - 1]], dtype=torch.int32, device=cuda_device)
    ends = torch.tensor([2, 4], dtype=torch.int32, device=cuda_device)
    r = routing.Routing(torch.ones(4, 2, device=cuda_device), rows, ends, rows, rows.reshape(-1))
    x = torch.arange(1, 5, device=cuda_device, dtype=torch.float32)[:, None].expand(4, 8).contiguous()
    sent = routing.dispatch_tokens(x, r)
    assert sent[:, 0].tolist() == [1, 2, 3, 4, 0, 0, 0, 0]
    y = torch.arange(1, 9, device=cuda_device, dtype=torch.float32)[:, None].expand(8, 8).contiguous().requires_grad_()
    routing.combine_tokens(y, r).sum().backward()
    assert y.grad[:, 0].tolist() == [1, 1, 1, 1, 0, 0, 0, 0]
    no_tokens = routing.Routing(torch.ones(0, 2, device=cuda_device), rows[:0], ends, rows[:0], rows[:0].reshape(-1))
    assert routing.dispatch_tokens(x[:0], no_tokens).shape == (0, 8) and routing.combine_tokens(x[:0], no_tokens).shape == (0, 8)


@pytest.mark.parametrize("end", [3, 0, -7, 100])
def test_places_past_the_last_end_count_as_none(cuda_device, end):
    """A routing that was not made by route_tokens: the last end decides which places are in use, in every pass alike; an end
    past all places counts as their number, one below none as none."""
    rows = torch.tensor([[0, 5], [4, 1], [2, 3]], dtype=torch.int32, device=cuda_device)
    ends = torch.tensor([1, end], dtype=torch.int32, device=cuda_device)
    weights = torch.full((3, 2), 2.0, device=cuda_device, requires_grad=True)
    r = routing.Routing(weights, rows, ends, rows, rows.reshape(-1))
    used = [max(0, min(6, end)) > place for place in range(6)]
    x = torch.tensor([[1.0], [2.0], [3.0]], device=cuda_device).expand(3, 8).contiguous().requires_grad_()
    sent = routing.dispatch_tokens(x, r)
    assert sent[:, 0].tolist() == [v * u for v, u in zip([1, 2, 3, 3, 2, 1], used)]
    taken = [[used[p] for p in token] for token in rows.tolist()]
    (dx,) = torch.autograd.grad(sent.sum(), x)
    assert dx[:, 0].tolist() == [sum(t) for t in taken]
    y = torch.arange(1.0, 7, device=cuda_device)[:, None].expand(6, 8).contiguous().requires_grad_()
    out = routing.combine_tokens(y, r)
    assert out[:, 0].tolist() == [sum(2 * (p + 1) * u for p, u in zip(*both)) for both in zip(rows.tolist(), taken)]
    dy, dweights = torch.autograd.grad(out.sum(), (y, weights))
    assert dy[:, 0].tolist() == [2 * u for u in used]
    assert dweights.tolist() == [[8 * (p + 1) * u for p, u in zip(*both)] for both in zip(rows.tolist(), taken)]


def test_offsets_beyond_32_bits(cuda_device):
    """Rows that end more than 2^32 bytes into their tensors."""
    if torch.cuda.get_device_properties(cuda_device).total_memory < 60e9:
        pytest.skip("needs 30 GB")
    tokens, top_k, hidden = 70000, 8, 4096
    r = routing.route_tokens(torch.randn(tokens, 16, device=cuda_device, generator=torch.Generator(cuda_device).manual_seed(0)), top_k)
    x = torch.randn(tokens, hidden, device=cuda_device, generator=torch.Generator(cuda_device).manual_seed(1)).bfloat16()
    sent = routing.dispatch_tokens(x, r)
    assert sent.numel() > 2 ** 31
    for part in (slice(0, 300), slice(-300, None)):
        assert torch.equal(sent[part], x[r.source[part].long() // top_k])
    y = sent.requires_grad_()
    back = routing.combine_tokens(y, r)
    assert ((back.float() - x.float()).abs() <= x.float().abs() * (2.0 ** -8 + 1e-5)).all()  # a token's weights add up to one
    (dy,) = torch.autograd.grad(back, y, x)
    for part in (slice(0, 300), slice(-300, None)):
        want = x[r.source[part].long() // top_k].double() * r.weights.reshape(-1)[r.source[part].long()].double()[:, None]
        assert ((dy[part].double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -23) + R.TINY["bfloat16"]).all()


# ------------------------------------------------------------- streams, graphs, same bits
def test_same_bits_on_every_run(cuda_device):
    logits = normal_logits(3000, 64, torch.bfloat16, cuda_device)
    first = routing.route_tokens(logits, 6, scoring="sigmoid", groups=8, top_groups=4, group_score="top2")
    y = normal_logits(18000, 264, torch.bfloat16, cuda_device)
    back = routing.combine_tokens(y, first)
    for _ in range(10):
        again = routing.route_tokens(logits, 6, scoring="sigmoid", groups=8, top_groups=4, group_score="top2")
        for f in ("weights", "experts", "ends", "rows", "source"):
            assert torch.equal(getattr(first, f), getattr(again, f))
        assert torch.equal(routing.combine_tokens(y, again), back)


def test_captured_graphs_replay_and_streams(cuda_device):
    graphs = []
    for tokens in (50, 2000):
        logits = normal_logits(tokens, 40, torch.bfloat16, cuda_device)
        x = normal_logits(tokens, 136, torch.bfloat16, cuda_device, seed=1)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r = routing.route_tokens(logits, 4)
            back = routing.combine_tokens(routing.dispatch_tokens(x, r), r)
        graphs.append((graph, logits, x, r, back))
    side = torch.cuda.Stream()
    for turn in range(3):
        for _, logits, *_ in graphs:
            logits.copy_(normal_logits(*logits.shape, torch.bfloat16, cuda_device, seed=turn))
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, logits, x, r, back in graphs:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                again = routing.route_tokens(logits, 4)
                other = routing.combine_tokens(routing.dispatch_tokens(x, again), again)
            torch.cuda.current_stream().wait_stream(side)
            assert torch.equal(r.source, again.source) and torch.equal(r.weights, again.weights) and torch.equal(back, other)
            # a token's copies weigh one in all
            assert ((back.float() - x.float()).abs() <= x.float().abs() * (2.0 ** -8 + 1e-6)).all()


def test_bad_arguments_are_refused(cuda_device):
    logits = torch.zeros(6, 16, device=cuda_device)
    route = routing.route_tokens
    for call, match in ((lambda: route(logits.double(), 2), "float64"), (lambda: route(logits[0], 2), "tokens, experts"), (lambda: route(logits, 0), "1 to 32 experts"),
                        (lambda: route(logits, 17), "no more than"), (lambda: route(torch.zeros(2, 1025, device=cuda_device), 2), "1 to 1024"),
                        (lambda: route(torch.zeros(2, 64, device=cuda_device), 33), "1 to 32 experts"), (lambda: route(logits, 2, scoring="relu"), "softmax or sigmoid"),
                        (lambda: route(logits, 2, group_score="mean"), "max or top2"), (lambda: route(logits, 2, groups=3, top_groups=1), "equally many"),
                        (lambda: route(logits, 2, groups=0), "groups"), (lambda: route(logits, 2, groups=4, top_groups=5), "1 to all groups"),
                        (lambda: route(logits, 5, groups=4, top_groups=1), "fewer experts"), (lambda: route(logits, 2, bias=torch.zeros(16, device=cuda_device).double()), "bias"),
                        (lambda: route(logits, 2, bias=torch.zeros(15, device=cuda_device)), "bias"), (lambda: route(logits, 2, bias=torch.zeros(16)), "bias"),
                        (lambda: route(logits, 2, mask=torch.ones(5, dtype=torch.bool, device=cuda_device)), "mask"),
                        (lambda: route(logits, 2, mask=torch.ones(6, device=cuda_device)), "mask")):
        with pytest.raises(ValueError, match=match):
            call()
    r = route(logits, 2)
    x = torch.zeros(6, 32, device=cuda_device)
    wrong = routing.Routing(r.weights[:3], r.experts, r.ends, r.rows, r.source)
    long = routing.Routing(r.weights, r.experts, r.ends, r.rows.long(), r.source)
    for call, match in ((lambda: routing.dispatch_tokens(x[:5], r), "6 rows"), (lambda: routing.dispatch_tokens(x.int(), r), "int32"),
                        (lambda: routing.dispatch_tokens(x[:, :0], r), "values"), (lambda: routing.combine_tokens(x, r), "12 rows"),
                        (lambda: routing.combine_tokens(x.repeat(2, 1), wrong), "weights"), (lambda: routing.dispatch_tokens(x, long), "int32"),
                        (lambda: routing.dispatch_tokens(x.cpu(), r), "CUDA")):
        with pytest.raises(ValueError, match=match):
            call()
    with torch.autograd.forward_ad.dual_level():
        make = torch.autograd.forward_ad.make_dual
        for call in (lambda: route(make(logits, logits), 2), lambda: routing.dispatch_tokens(make(x, x), r),
                     lambda: routing.combine_tokens(make(x, x).repeat(2, 1), r)):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
    # what a backward pass needs may not change before it
    leaf = logits.clone().requires_grad_()
    r = route(leaf, 2)
    y = torch.ones(12, 8, device=cuda_device, requires_grad=True)
    out = routing.combine_tokens(y, r)
    r.rows.add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
