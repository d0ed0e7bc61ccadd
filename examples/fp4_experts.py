"""A layer of FP4 experts from dense weights to a gradient: quantise, merge an adapter, route, multiply, differentiate.

    python examples/fp4_experts.py --experts 8 --tokens 512 --hidden 1024 --inner 2816 --format nvfp4

1. the experts' dense weights become one packed stack (``fp4.quantize_nvfp4`` / ``fp4.quantize_mxfp4``);
2. a LoRA update is merged into one expert in place (``transform.merge_lora``), which changes the stack;
3. tokens are sorted by expert and go through up and down projections (``fp4.grouped_linear_fp4``), with the ends of
   the groups staying on the device;
4. a loss is differentiated back to the tokens through the frozen packed weights.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from piper_offload_b200 import fp4, transform  # noqa: E402


def sort_by_expert(router: torch.Tensor, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(order of the tokens, int32 ends of the experts' groups): each token goes to its best expert."""
    expert = (x @ router.T).argmax(dim=1)
    return expert.argsort(stable=True), torch.bincount(expert, minlength=router.shape[0]).cumsum(0).to(torch.int32)


def experts_forward(x, order, ends, up, down):
    """Every token through its expert's two projections, in the tokens' own order."""
    inner = torch.nn.functional.silu(fp4.grouped_linear_fp4(x[order], up, ends))
    y = fp4.grouped_linear_fp4(inner, down, ends)
    return torch.empty_like(y).index_copy(0, order, y)


def run(experts: int, tokens: int, hidden: int, inner: int, fmt: str, rank: int = 16, seed: int = 0) -> dict[str, float]:
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).bfloat16()

    quantize = fp4.quantize_nvfp4 if fmt == "nvfp4" else fp4.quantize_mxfp4
    dense_up, dense_down = normal(experts, inner, hidden, std=hidden ** -0.5), normal(experts, hidden, inner, std=inner ** -0.5)
    up, down = quantize(dense_up, swizzled=True), quantize(dense_down, swizzled=True)
    packed = fp4.dequantize_fp4(up)
    quantisation_error = float((packed - dense_up).float().norm() / dense_up.float().norm())

    # an adapter for expert 1's up projection, merged where the stack holds it
    a, b = normal(rank, hidden, std=0.05), normal(inner, rank, std=0.05)
    transform.merge_lora({"experts.1.up": up.expert(1)}, [({"experts.1.up": (a, b)}, 1.0)], stochastic_rounding=False)
    merged = fp4.dequantize_fp4(up).float()
    wanted = packed[1].float() + b.float() @ a.float()
    merge_error = float((merged[1] - wanted).norm() / wanted.norm())
    untouched = float((merged - packed)[torch.arange(experts, device="cuda") != 1].abs().max())

    router, x = normal(experts, hidden), normal(tokens, hidden)
    order, ends = sort_by_expert(router, x)
    x.requires_grad_()
    y = experts_forward(x, order, ends, up, down)
    y.float().square().mean().backward()

    # the same layer with dense weights of the packed values and unquantised tokens
    wu, wd = fp4.dequantize_fp4(up).float(), fp4.dequantize_fp4(down).float()
    expert = torch.searchsorted(ends, torch.arange(tokens, device="cuda", dtype=torch.int32), right=True)
    want = torch.empty_like(y, dtype=torch.float32)
    for e in range(experts):
        rows = order[expert == e]
        want[rows] = torch.nn.functional.silu(x.detach()[rows].float() @ wu[e].T) @ wd[e].T
    return {"quantisation_error": quantisation_error, "merge_error": merge_error, "largest_change_elsewhere": untouched,
            "output_error": float((y.detach().float() - want).norm() / want.norm()), "gradient_norm": float(x.grad.float().norm())}


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--experts", type=int, default=8)
    ap.add_argument("--tokens", type=int, default=512)
    ap.add_argument("--hidden", type=int, default=1024)
    ap.add_argument("--inner", type=int, default=2816)
    ap.add_argument("--format", choices=("nvfp4", "mxfp4"), default="nvfp4")
    args = ap.parse_args()
    for name, value in run(args.experts, args.tokens, args.hidden, args.inner, args.format).items():
        print(f"{name:26s} {value:.4g}")


if __name__ == "__main__":
    main()
