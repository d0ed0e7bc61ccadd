"""CPU: what the differentiable FP4 products keep of a weight for the backward pass, with the kernels' calls replaced by
dense products over the codes."""

from __future__ import annotations

import pytest
import torch

from piper_offload_b200 import fp4
from piper_offload_b200 import weights as W


def values(w) -> torch.Tensor:
    """A stand-in for a weight's values in which each of its parts counts."""
    v = w.qdata.float() * w.scale.view(torch.uint8).float().sum() * (2.0 if w.is_swizzled_scales else 1.0)
    second = getattr(w, "per_tensor_scale", None)
    return v if second is None else v * second.sum()


@pytest.fixture(autouse=True)
def dense_calls(monkeypatch):
    monkeypatch.setattr(fp4, "_linear", lambda x, w, ends, act: x @ values(w)[-1 if ends is not None else ...].T)
    monkeypatch.setattr(fp4, "_grad_input", lambda g, w, ends: g @ values(w)[-1 if ends is not None else ...])
    monkeypatch.setattr(fp4, "_check_ends", lambda *args: None)


def weight(kind):
    g = torch.Generator().manual_seed(4)
    lead = (2,) if kind in ("mx stack", "nv stack") else ()
    q = torch.randint(0, 256, (*lead, 8, 16), dtype=torch.uint8, generator=g)
    if kind.startswith("mx"):
        s = torch.randint(1, 9, (*lead, 8, 1), dtype=torch.uint8, generator=g)
        return (W.MXExperts if lead else W.MXWeight)(q, s, torch.float4_e2m1fn_x2)
    s = torch.randint(1, 9, (*lead, 8, 2), dtype=torch.uint8, generator=g).view(torch.float8_e4m3fn)
    return (W.NVFP4Experts if lead else W.NVFP4Weight)(q, s, torch.ones(lead or (1,)))


KINDS = ["mx", "nv", "mx stack", "nv stack"]


def forward(w, ends=torch.tensor([1, 3], dtype=torch.int32)):
    x = torch.ones((3, 16), requires_grad=True)
    return x, fp4.grouped_linear_fp4(x, w, ends) if w.qdata.ndim == 3 else fp4.linear_fp4(x, w)


@pytest.mark.parametrize("kind", KINDS)
def test_parts_put_in_place_of_others_leave_the_gradient_alone(kind):
    names = ["qdata", "scale", "is_swizzled_scales"] + ["per_tensor_scale"] * kind.startswith("nv")
    w = weight(kind)
    x, y = forward(w)
    y.sum().backward()
    want = x.grad
    for name in names:
        w = weight(kind)
        x, y = forward(w)
        old = getattr(w, name)
        setattr(w, name, not old if isinstance(old, bool) else old.view(torch.uint8).add(1).view(old.dtype) if name != "per_tensor_scale" else old * 3)
        y.sum().backward()
        assert torch.equal(x.grad, want), name


@pytest.mark.parametrize("kind", KINDS)
def test_parts_changed_by_torch_are_noticed(kind):
    for name in ["qdata", "scale"] + ["per_tensor_scale"] * kind.startswith("nv"):
        w = weight(kind)
        _, y = forward(w)
        t = getattr(w, name)
        (t if t.dtype is torch.float32 else t.view(torch.uint8)).add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            y.sum().backward()


@pytest.mark.parametrize("kind", KINDS)
def test_saved_tensor_hooks_see_no_weight(kind):
    """Hooks that move saved tensors away (to the host, say) would move a frozen weight that stays in use."""
    w, packed = weight(kind), []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(t) or t.clone(), lambda t: t):
        x, y = forward(w)
    own = {t.data_ptr() for t in (w.qdata, w.scale, getattr(w, "per_tensor_scale", None)) if t is not None}
    assert not own & {t.data_ptr() for t in packed}
    y.sum().backward()
    again, z = forward(w)
    z.sum().backward()
    assert torch.equal(x.grad, again.grad)


@pytest.mark.parametrize("kind", KINDS)
def test_weights_made_in_inference_mode(kind):
    with torch.inference_mode():
        frozen = weight(kind)
    x, y = forward(frozen)
    y.sum().backward()
    again, z = forward(weight(kind))
    z.sum().backward()
    assert torch.equal(x.grad, again.grad)


def test_two_backward_passes_give_twice_the_gradient():
    x, y = forward(weight("nv"))
    y.sum().backward(retain_graph=True)
    once = x.grad.clone()
    y.sum().backward()
    assert torch.equal(x.grad, 2 * once)
