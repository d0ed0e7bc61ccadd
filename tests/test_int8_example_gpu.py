"""GPU: the INT8 experts' example runs, and its results and gradients are those of a dense layer of the same values; the
operators together in a graph that is captured and replayed."""

from __future__ import annotations

import os
import subprocess
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

import int8_experts as example  # noqa: E402
from piper_offload_b200 import fp4, int8, routing  # noqa: E402

pytestmark = pytest.mark.gpu

# A token's codes are off by up to half a unit of max|x| / 127: of normal values about 0.75 % of their norm, once for each of
# two projections (of the second's SiLU more, whose values have a longer tail), and bf16 rounds by up to 0.4 % six times.
CLOSE = 0.05


@pytest.mark.parametrize("sizes", [(16, 4, 200, 256, 336), (5, 2, 33, 144, 100), (8, 1, 1, 64, 48)])
def test_example(sizes, cuda_device):
    out = example.run(*sizes)
    assert out["largest_change_elsewhere"] == 0 and out["choices"] == sizes[1] * sizes[2]
    assert out["merge_error"] < 0.02  # half a unit of max|w| / 127 of normal values, as of tokens, and a bf16 scale
    for name in ("output_error", "token_gradient_error") + (("router_gradient_error",) if sizes[1] > 1 else ()):
        assert out[name] < CLOSE, name


def test_command(cuda_device):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "int8_experts.py")
    done = subprocess.run([sys.executable, path, "--experts", "4", "--top-k", "2", "--tokens", "40", "--hidden", "128", "--inner", "96"],
                          capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "output_error" in done.stdout, done.stderr


def test_layer_in_a_graph(cuda_device):
    """Routing, exchange and both projections captured once and replayed on other tokens, which go to other experts."""
    g = torch.Generator(cuda_device).manual_seed(0)
    up, down = (example.pack(torch.randn(shape, generator=g, device=cuda_device).bfloat16()) for shape in ((6, 80, 128), (6, 128, 80)))
    router = torch.randn(6, 128, generator=g, device=cuda_device).bfloat16()
    x = torch.randn(70, 128, generator=g, device=cuda_device).bfloat16()
    with torch.no_grad():
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            example.layer(x, router, up, down, 2)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, r = example.layer(x, router, up, down, 2)
        for _ in range(3):
            x.copy_(torch.randn(70, 128, generator=g, device=cuda_device))
            graph.replay()
            again, s = example.layer(x, router, up, down, 2)
            assert torch.equal(y, again) and torch.equal(r.source, s.source)


def test_training_step_in_a_graph(cuda_device):
    """The layer with its gradients, captured once and replayed on other tokens and logits: the eager step's bits."""
    g = torch.Generator(cuda_device).manual_seed(1)
    up, down = (example.pack(torch.randn(shape, generator=g, device=cuda_device).bfloat16()) for shape in ((6, 80, 128), (6, 128, 80)))
    x, dy = (torch.randn(300, 128, generator=g, device=cuda_device).bfloat16() for _ in range(2))
    logits = torch.randn(300, 6, generator=g, device=cuda_device)
    x.requires_grad_(), logits.requires_grad_()

    def step():
        r = routing.route_tokens(logits, 2, scoring="sigmoid", bias=logits.detach()[0].clone())
        h = int8.grouped_linear_int8(routing.dispatch_tokens(x, r), up, r.ends)
        y = routing.combine_tokens(int8.grouped_linear_int8(h, down, r.ends), r)
        return y.detach(), *torch.autograd.grad(y, (x, logits), dy)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(300, 128, generator=g, device=cuda_device))
            logits.copy_(torch.randn(300, 6, generator=g, device=cuda_device))
        graph.replay()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)


def test_routing_feeds_the_fp4_products_too(cuda_device):
    g = torch.Generator(cuda_device).manual_seed(0)
    dense = torch.randn(5, 96, 128, generator=g, device=cuda_device).bfloat16()
    x = torch.randn(40, 128, generator=g, device=cuda_device).bfloat16()
    w = fp4.quantize_nvfp4(dense, swizzled=True)
    r = routing.route_tokens(torch.randn(40, 5, generator=g, device=cuda_device), 2, mask=torch.arange(40, device=cuda_device) > 3)
    y = fp4.grouped_linear_fp4(routing.dispatch_tokens(x, r), w, r.ends)
    packed = example.pack(dense)
    z = int8.grouped_linear_int8(routing.dispatch_tokens(x, r), packed, r.ends)
    back, other = routing.combine_tokens(y, r), routing.combine_tokens(z, r)
    assert not back[:4].any() and not other[:4].any()
    # 4 bits against 8 of the same values: e2m1's steps are up to a third of a value, a tenth of the norm for each operand
    assert (back.float() - other.float()).norm() < 0.3 * other.float().norm()
