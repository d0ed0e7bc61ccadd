"""A layer of INT8 experts from a router's logits to gradients: route, merge an adapter, exchange, multiply, differentiate.

    python examples/int8_experts.py --experts 16 --top-k 4 --tokens 512 --hidden 1024 --inner 1408

1. the experts' dense weights become int8 codes with a scale for each row, stacked (``weights.Int8Experts``);
2. a LoRA update is merged into one expert in place (``transform.merge_lora``), which changes the stack;
3. a router's logits choose each token's experts (``routing.route_tokens``); tokens are copied to their places
   (``routing.dispatch_tokens``), go through up and down projections (``int8.grouped_linear_int8``) and are added up again
   by the router's weights (``routing.combine_tokens``); nothing of it is read by the host;
4. a loss is differentiated back to the tokens, through the frozen packed weights, and to the router.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from piper_offload_b200 import int8, routing, transform, weights  # noqa: E402


def pack(dense: torch.Tensor) -> weights.Int8Experts:
    """Codes and bf16 scales of each row of a stack (experts, rows, cols)."""
    scale = (dense.float().abs().amax(-1, keepdim=True).clamp_min(1e-12) / 127).bfloat16()
    codes = torch.round(dense.float() / scale.float()).clamp(-127, 127).to(torch.int8)
    return weights.Int8Experts(codes, scale, (1, dense.shape[-1]))


def values(stack: weights.Int8Experts) -> torch.Tensor:
    return stack.qdata.float() * stack.scale.float()


def layer(x, router, up, down, top_k):
    """Every token through its experts' two projections, and the routing."""
    r = routing.route_tokens(x @ router.T, top_k, scoring="sigmoid")
    h = torch.nn.functional.silu(int8.grouped_linear_int8(routing.dispatch_tokens(x, r), up, r.ends))
    return routing.combine_tokens(int8.grouped_linear_int8(h, down, r.ends), r), r


def dense_layer(x, router, up, down, chosen, top_k):
    """The same with dense weights, unquantised tokens and the experts that were chosen."""
    score = torch.sigmoid(x @ router.T).gather(1, chosen)
    w = score / score.sum(1, keepdim=True)
    y = torch.zeros_like(x)
    for j in range(top_k):
        e = chosen[:, j]
        h = torch.nn.functional.silu(torch.einsum("th,tih->ti", x, up[e]))
        y = y + w[:, j:j + 1] * torch.einsum("ti,thi->th", h, down[e])
    return y


def run(experts: int, top_k: int, tokens: int, hidden: int, inner: int, rank: int = 16, seed: int = 0) -> dict[str, float]:
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).bfloat16()

    up, down = pack(normal(experts, inner, hidden, std=hidden ** -0.5)), pack(normal(experts, hidden, inner, std=inner ** -0.5))
    before = values(up)
    a, b = normal(rank, hidden, std=0.05), normal(inner, rank, std=0.05)
    transform.merge_lora({"experts.1.up": up.expert(1)}, [({"experts.1.up": (a, b)}, 1.0)], stochastic_rounding=False)
    merged, wanted = values(up), before[1] + b.float() @ a.float()
    elsewhere = torch.arange(experts, device="cuda") != 1

    x, router = normal(tokens, hidden).requires_grad_(), normal(experts, hidden, std=hidden ** -0.5).requires_grad_()
    y, r = layer(x, router, up, down, top_k)
    upstream = normal(tokens, hidden)
    y.backward(upstream)

    x64, router64 = (t.detach().float().requires_grad_() for t in (x, router))
    want = dense_layer(x64, router64, merged, values(down), r.experts.long(), top_k)
    want.backward(upstream.float())

    def error(got, exact):
        return float((got.detach().float() - exact).norm() / exact.norm())

    return {"merge_error": error(merged[1], wanted), "largest_change_elsewhere": float((merged - before)[elsewhere].abs().max()),
            "output_error": error(y, want.detach()), "token_gradient_error": error(x.grad, x64.grad),
            "router_gradient_error": error(router.grad, router64.grad), "choices": int(r.ends[-1])}


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--experts", type=int, default=16)
    ap.add_argument("--top-k", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=512)
    ap.add_argument("--hidden", type=int, default=1024)
    ap.add_argument("--inner", type=int, default=1408)
    args = ap.parse_args()
    for name, value in run(args.experts, args.top_k, args.tokens, args.hidden, args.inner).items():
        print(f"{name:26s} {value:.4g}")


if __name__ == "__main__":
    main()
