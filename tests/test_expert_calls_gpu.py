"""GPU: the calls that compiled code makes and those that it declines are the same; what autograd asks of both."""

from __future__ import annotations

import pytest
import torch

import test_int8_gpu as T
from piper_offload_b200 import _native_calls, int8, routing
from piper_offload_b200 import _native_int8 as nat

pytestmark = pytest.mark.gpu


class Declines:
    def __getattr__(self, name):
        return lambda *args: None


@pytest.fixture
def declined(monkeypatch):
    """Every call takes the path that is written in Python."""
    monkeypatch.setattr(int8, "calls", Declines)
    monkeypatch.setattr(routing, "calls", Declines)


@pytest.fixture(autouse=True)
def device_status_clean(cuda_device):
    yield
    assert nat.device_status(cuda_device) == 0, "a bounded device wait timed out"


def layer(device, seed=0):
    """One of everything, forward and backward: the outputs and gradients in order."""
    w, _, _ = T.make_weight("zero", 96, 64, device, experts=4)
    one, _, _ = T.make_weight("bnb8", 64, 96, device)
    g = torch.Generator(device).manual_seed(seed)
    x = torch.randn(40, 64, generator=g, device=device).half().requires_grad_()
    logits = torch.randn(40, 4, generator=g, device=device).requires_grad_()
    mask = torch.rand(40, generator=g, device=device) < 0.8
    r = routing.route_tokens(logits, 2, mask=mask, bias=torch.linspace(0, 0.1, 4, device=device), scoring="sigmoid")
    h = int8.grouped_linear_int8(routing.dispatch_tokens(x, r), w, r.ends)
    y = routing.combine_tokens(int8.linear_int8(h, one), r)
    y.float().square().sum().backward()
    return [r.weights, r.experts, r.ends, r.rows, r.source, h, y, x.grad, logits.grad,
            int8.grouped_linear_int8_grad_input(h.detach(), w, r.ends), int8.linear_int8_grad_input(y.detach(), one)]


def test_both_paths_give_the_same(cuda_device, monkeypatch):
    compiled = layer(cuda_device)
    launched = nat.launches()
    monkeypatch.setattr(int8, "calls", Declines)
    monkeypatch.setattr(routing, "calls", Declines)
    written = layer(cuda_device)
    assert nat.launches() > launched
    for a, b in zip(compiled, written):
        assert a.dtype is b.dtype and torch.equal(a, b) and a.requires_grad == b.requires_grad


def test_the_path_written_in_python(declined, cuda_device):
    T.test_product(33, 70, 208, torch.bfloat16, cuda_device)
    T.test_gradient(33, 70, 208, torch.bfloat16, cuda_device)
    T.test_kinds_of_weights(2, "quanto scalar", cuda_device)
    T.test_groups([9, 5, 30, 20], "zero", cuda_device)
    T.test_grouped_backward_and_frozen_weights(cuda_device)
    T.test_strides_and_alignment(torch.float16, cuda_device)
    T.test_no_tokens(cuda_device)


def test_plain_calls_are_compiled(cuda_device):
    w, _, _ = T.make_weight("zero", 96, 64, cuda_device)
    x = torch.randn(5, 64, device=cuda_device)
    calls = _native_calls.calls()
    assert calls.int8(x, w, None, False) is not None and calls.int8(x[:, :63], w, None, False) is None
    assert calls.route(x, 2, 0, None, 1, 1, 0, True, 1.0, None) is not None
    r = routing.route_tokens(x, 2)
    assert calls.dispatch(x, r.rows, r.ends) is not None and calls.dispatch(x[:4], r.rows, r.ends) is None
    assert calls.combine(torch.cat((x, x)), r.weights, r.rows, r.ends) is not None


@pytest.mark.parametrize("path", ["compiled", "written"])
def test_gradients_are_not_differentiable(path, cuda_device, request):
    if path == "written":
        request.getfixturevalue("declined")
    w, _, _ = T.make_weight("rows", 96, 64, cuda_device)
    x = torch.randn(6, 64, device=cuda_device, requires_grad=True)
    logits = torch.randn(6, 8, device=cuda_device, requires_grad=True)
    r = routing.route_tokens(logits, 2)
    rows = torch.randn(12, 64, device=cuda_device, requires_grad=True)
    for out, leaf in ((int8.linear_int8(x, w), x), (r.weights, logits), (routing.dispatch_tokens(x, r), x), (routing.combine_tokens(rows, r), rows)):
        upstream = torch.randn(out.shape, device=cuda_device, requires_grad=True)
        (g,) = torch.autograd.grad(out, leaf, upstream, create_graph=True)
        assert g.shape == leaf.shape
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()
    # a graph of the gradients that nothing is asked of is fine, and without one they are plain
    out = int8.linear_int8(x, w)
    (g,) = torch.autograd.grad(out, x, torch.ones_like(out), create_graph=True)
    assert not g.requires_grad


@pytest.mark.parametrize("path", ["compiled", "written"])
def test_what_needs_a_gradient(path, cuda_device, request):
    if path == "written":
        request.getfixturevalue("declined")
    logits = torch.randn(6, 8, device=cuda_device, requires_grad=True)
    r = routing.route_tokens(logits, 2)
    assert r.weights.requires_grad and not any(t.requires_grad for t in (r.experts, r.ends, r.rows, r.source))
    with torch.no_grad():
        assert not routing.route_tokens(logits, 2).weights.requires_grad
    plain = routing.route_tokens(logits.detach(), 2)
    y = torch.randn(12, 16, device=cuda_device)
    assert not routing.combine_tokens(y, plain).requires_grad and routing.combine_tokens(y, r).requires_grad
    # only the weights' gradient is wanted, and it reaches the logits
    routing.combine_tokens(y, r).sum().backward()
    assert logits.grad is not None and logits.grad.isfinite().all()
    # a result that is not used in the end asks for nothing
    x = torch.randn(6, 16, device=cuda_device, requires_grad=True)
    routing.dispatch_tokens(x, r)
    (x * 2).sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, 2))
    with torch.inference_mode():
        assert torch.equal(routing.dispatch_tokens(x, plain), routing.dispatch_tokens(x.clone(), plain))


def test_results_of_a_routing_are_tensors_of_their_own(cuda_device):
    logits = torch.randn(9, 8, device=cuda_device)
    r = routing.route_tokens(logits, 3)
    rows, version = r.rows.clone(), r.rows._version
    r.experts.fill_(-7)
    r.weights.zero_()
    assert torch.equal(r.rows, rows) and r.rows._version == version and not r.rows._is_view()
    assert r.weights.is_contiguous() and r.ends.shape == (8,) and r.source.shape == (27,)


def test_calls_from_two_threads(cuda_device):
    """Two threads on streams of their own, forward and backward: what one does is none of the other's."""
    import threading

    want = [layer(cuda_device, seed) for seed in (1, 2)]
    got, failed = [[], []], []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(8):
                    got[i] = layer(cuda_device, i + 1)
            stream.synchronize()
        except Exception as exc:  # noqa: BLE001
            failed.append(exc)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for a, b in zip(want[0] + want[1], got[0] + got[1]):
        assert torch.equal(a, b)
