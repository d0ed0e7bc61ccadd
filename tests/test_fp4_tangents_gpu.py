"""GPU: the FP4 operators under forward-mode differentiation, which they have no formula for: refused, not dropped."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from piper_offload_b200 import fp4

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["mxfp4", "nvfp4"])
def weights(request, cuda_device):
    """One weight, a stack of two, and the ends of their rows."""
    dense = torch.randn((2, 48, 64), generator=torch.Generator(cuda_device).manual_seed(1), device=cuda_device).bfloat16()
    quantize = fp4.quantize_mxfp4 if request.param == "mxfp4" else fp4.quantize_nvfp4
    return quantize(dense[0]), quantize(dense), torch.tensor([3, 5], dtype=torch.int32, device=cuda_device)


def calls(one, stack, ends):
    """Each operator that differentiates or is a derivative, with the width of its input."""
    return [(64, lambda t: fp4.linear_fp4(t, one)), (64, lambda t: fp4.grouped_linear_fp4(t, stack, ends)),
            (48, lambda t: fp4.linear_fp4_grad_input(t, one)), (48, lambda t: fp4.grouped_linear_fp4_grad_input(t, stack, ends))]


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_tangents_are_refused(weights, dtype, requires_grad, cuda_device):
    for width, call in calls(*weights):
        x = torch.ones((5, width), dtype=dtype, device=cuda_device, requires_grad=requires_grad)
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(x, torch.ones_like(x))
            for t in (dual, dual[:, :]):  # itself and a view that carries the tangent on
                with pytest.raises(ValueError, match="forward-mode"):
                    call(t)
                with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                    call(t)
            # a tensor without a tangent is taken inside a level, a dual's primal too
            want = call(x.detach())
            assert torch.equal(call(forward_ad.unpack_dual(dual).primal.detach()), want)
        assert torch.equal(call(x), want)


def test_tangents_of_the_second_level_are_refused(cuda_device):
    w = fp4.quantize_nvfp4(torch.ones((48, 64), dtype=torch.bfloat16, device=cuda_device))
    x, act = torch.ones((5, 64), device=cuda_device), torch.full((1,), 0.01, device=cuda_device)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(act, torch.ones_like(act))
        with pytest.raises(ValueError, match="forward-mode"):
            fp4.linear_fp4(x, w, act_per_tensor_scale=dual)
    assert fp4.linear_fp4(x, w, act_per_tensor_scale=act).isfinite().all()


def test_functional_jvp_is_refused(weights, cuda_device):
    for width, call in calls(*weights):
        x = torch.ones((5, width), device=cuda_device)
        with pytest.raises((ValueError, RuntimeError)):
            torch.func.jvp(call, (x,), (torch.ones_like(x),))
