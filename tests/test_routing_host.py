"""CPU: the routing library loads, exports what its header declares, and refuses bad arguments before touching a device; the
reference of the GPU tests is checked against torch."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import numpy as np
import pytest
import torch

import routing_reference as R
from piper_offload_b200 import _native_routing as nat
from piper_offload_b200 import routing

HEADER = Path(__file__).resolve().parents[1] / "include" / "piper_routing.h"


def test_library_exports_what_the_header_declares():
    names = set(re.findall(r"\b(piper_routing_\w+)\s*\(", HEADER.read_text()))
    assert names == set(nat.EXPORTED_SYMBOLS)
    for name in names:
        assert hasattr(nat.load(), name), name
    assert "sm_100a" in nat.version()


def config(**kw) -> nat.Config:
    fields = {"tokens": 8, "experts": 16, "top_k": 2, "scoring": 0, "groups": 1, "top_groups": 1, "group_score": 0, "renormalize": 1,
              "scale": 1.0}
    return nat.Config(**{**fields, **kw})


BAD_CONFIGS = [({"experts": 0}, "1 to 1024"), ({"experts": 1025}, "1 to 1024"), ({"top_k": 0}, "1 to 32"), ({"top_k": 17}, "no more than"),
               ({"experts": 64, "top_k": 33}, "1 to 32"), ({"tokens": -1}, "choices"), ({"tokens": 1 << 30}, "choices"), ({"scoring": 2}, "scoring"),
               ({"groups": 3}, "equally many"), ({"groups": 0}, "1 to 32 groups"), ({"groups": 4, "top_groups": 5}, "all groups"),
               ({"groups": 4, "top_groups": 0}, "all groups"), ({"groups": 8, "top_k": 3}, "fewer experts"), ({"group_score": 2}, "group score")]


def route(c: nat.Config, **kw) -> int:
    a = {"logits": 0x1000, "stride": 16, "dtype": 0, "bias": None, "mask": None, "weights": 0x2000, "experts": 0x3000, "ends": 0x4000,
         "rows": 0x5000, "source": 0x6000, "ws": None, "bytes": 0, **kw}
    return nat.load().piper_routing_route(ctypes.byref(c), *a.values(), None)


def route_grad(c: nat.Config, **kw) -> int:
    a = {"logits": 0x1000, "stride": 16, "dtype": 0, "experts": 0x3000, "grad": 0x4000, "dlogits": 0x5000, **kw}
    return nat.load().piper_routing_route_grad(ctypes.byref(c), *a.values(), None)


@pytest.mark.parametrize("change,match", BAD_CONFIGS, ids=lambda v: v if isinstance(v, str) else "-".join(map(str, v.items())))
def test_bad_configurations_are_refused(change, match):
    c, n = config(**change), ctypes.c_size_t()
    for call in (lambda: route(c), lambda: route_grad(c), lambda: nat.load().piper_routing_workspace(ctypes.byref(c), ctypes.byref(n))):
        with pytest.raises(ValueError, match=match):
            nat.check(call())


def test_bad_arguments_are_refused():
    c = config()
    for kw, match in (({"logits": None}, "null"), ({"weights": None}, "null"), ({"experts": None}, "null"), ({"ends": None}, "null"),
                      ({"rows": None}, "null"), ({"source": None}, "null"), ({"stride": 15}, "overlap"), ({"dtype": 3}, "bfloat16"),
                      ({"logits": 0x1001}, "aligned")):
        with pytest.raises(ValueError, match=match):
            nat.check(route(c, **kw))
    for kw, match in (({"logits": None}, "null"), ({"experts": None}, "null"), ({"grad": None}, "null"), ({"dlogits": None}, "null"),
                      ({"stride": 3}, "overlap"), ({"dtype": -1}, "bfloat16"), ({"dlogits": 0x5001}, "aligned")):
        with pytest.raises(ValueError, match=match):
            nat.check(route_grad(c, **kw))
    many = config(tokens=100000)
    for kw in ({}, {"ws": 0x10000, "bytes": 64}, {"ws": 0x10002, "bytes": 1 << 30}):
        with pytest.raises(RuntimeError, match="workspace"):
            nat.check(route(many, **kw))


def test_workspace_is_for_many_tokens_only():
    n = ctypes.c_size_t()
    for tokens, least in ((0, 0), (1, 0), (64, 0), (100000, 16 * 4)):
        nat.check(nat.load().piper_routing_workspace(ctypes.byref(config(tokens=tokens)), ctypes.byref(n)))
        assert (n.value > 0) == (least > 0) and n.value >= least and n.value < 1 << 20


def exchange(**kw) -> nat.Exchange:
    fields = {"tokens": 8, "top_k": 2, "hidden": 64, "dtype": 0, "rows": 0x1000, "total": 0x2000}
    return nat.Exchange(**{**fields, **kw})


def exchange_calls(e: nat.Exchange, **kw):
    lib, ref = nat.load(), ctypes.byref(e)
    a = {"x": 0x10000, "stride": 64, "w": 0x30000, "out": 0x20000, "dout": 0x40000, "dw": 0x50000, **kw}
    yield lambda: lib.piper_routing_dispatch(ref, a["x"], a["stride"], a["out"], None)
    yield lambda: lib.piper_routing_combine(ref, a["x"], a["stride"], a["w"], a["out"], None)
    yield lambda: lib.piper_routing_combine_grad(ref, a["x"], a["stride"], a["w"], a["dout"], 64, a["out"], a["dw"], None)


@pytest.mark.parametrize("change,match", [({"dtype": 5}, "bfloat16"), ({"top_k": 0}, "1 to 32"), ({"top_k": 33}, "1 to 32"), ({"tokens": -1}, "choices"),
                                          ({"tokens": 1 << 30}, "choices"), ({"hidden": 0}, "values"), ({"hidden": 1 << 25}, "values"),
                                          ({"rows": None}, "null"), ({"total": None}, "null")])
def test_bad_exchanges_are_refused(change, match):
    for call in exchange_calls(exchange(**change)):
        with pytest.raises(ValueError, match=match):
            nat.check(call())


@pytest.mark.parametrize("change,match", [({"x": None}, "null"), ({"out": None}, "null"), ({"x": 0x10001}, "aligned"), ({"out": 0x20001}, "aligned"),
                                          ({"stride": -64}, "negative")])
def test_bad_exchange_arguments_are_refused(change, match):
    for call in exchange_calls(exchange(), **change):
        with pytest.raises(ValueError, match=match):
            nat.check(call())
    for change in ({"w": None}, {"dout": None}, {"dw": None}):
        with pytest.raises(ValueError, match="null"):
            nat.check(list(exchange_calls(exchange(), **change))[2]())


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="CUDA"):
        routing.route_tokens(torch.zeros(4, 8), 2)
    i = torch.zeros(4, 2, dtype=torch.int32)
    r = routing.Routing(torch.zeros(4, 2), i, i[0], i, i.reshape(-1))
    for call in (lambda: routing.dispatch_tokens(torch.zeros(4, 8), r), lambda: routing.combine_tokens(torch.zeros(8, 8), r)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


# ------------------------------------------------------------- the reference against torch
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_reference_weights_and_gradients_are_torchs(scoring, renormalize):
    g = np.random.default_rng(1)
    l64, grad = g.standard_normal((20, 12)), g.standard_normal((20, 3))
    weights, experts, ends, rows, source = R.route(l64, 3, scoring=scoring, renormalize=renormalize, scale=1.5)
    leaf = torch.from_numpy(l64).requires_grad_()
    score = torch.sigmoid(leaf) if scoring == "sigmoid" else torch.softmax(leaf, 1)
    top, at = score.topk(3, dim=1)
    want = (top / top.sum(1, keepdim=True) if renormalize else top) * 1.5
    np.testing.assert_array_equal(experts, at.numpy())
    np.testing.assert_allclose(weights, want.detach().numpy(), rtol=1e-12)
    want.backward(torch.from_numpy(grad))
    got, size = R.gradient(l64, experts, grad, scoring=scoring, renormalize=renormalize, scale=1.5)
    np.testing.assert_allclose(got, leaf.grad.numpy(), atol=1e-14)
    assert (size >= np.abs(got) * (1 - 1e-12)).all()
    flat = torch.from_numpy(experts).reshape(-1)
    np.testing.assert_array_equal(source, flat.argsort(stable=True).numpy())
    np.testing.assert_array_equal(ends, torch.bincount(flat, minlength=12).cumsum(0).numpy())
    np.testing.assert_array_equal(source[rows.reshape(-1)], np.arange(60))


def test_reference_groups_and_biases():
    logits = np.array([3.0, 0.0, 1.0, 2.9, -1.0, 2.0])
    assert R.choose(logits, 2) == [0, 3]
    assert R.choose(logits, 2, groups=3, top_groups=1) == [0, 1]
    assert R.choose(logits, 2, groups=3, top_groups=2) == [0, 3]
    # two best added up: {3, 0}, {1, 2.9}, {-1, 2} by their sigmoids
    assert R.choose(logits, 2, groups=3, top_groups=1, group_score="top2", scoring="sigmoid") == [3, 2]
    assert R.choose(logits, 2, bias=np.array([0, 5, 0, 0, 6, 0.0])) == [4, 1]
    closed = np.array([-np.inf, -np.inf, 1.0, -np.inf, np.nan, 2.0])
    assert R.choose(closed, 4) == [5, 2, 4, -1]
    assert R.choose(np.zeros(6), 3, groups=3, top_groups=2) == [0, 1, 2]
