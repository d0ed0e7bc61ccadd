"""From a router's logits to the experts' products and back, on sm_100a kernels of ``libpiper_routing.so``.

* :func:`route_tokens`: each token's experts, their weights, and the order of
  all choices by expert, as the grouped products (:mod:`~.fp4`, :mod:`~.int8`)
  take it;
* :func:`dispatch_tokens`: the tokens' rows copied to their places in that order;
* :func:`combine_tokens`: the experts' rows added up by the weights, token by
  token.

All three are differentiable (the weights with respect to the logits, the rows
and the weights of the exchange); the gradients are not differentiable
themselves, and inputs with a forward-mode tangent are refused. A layer of
experts is::

    r = routing.route_tokens(x @ router.T, 2)
    h = act(int8.grouped_linear_int8(routing.dispatch_tokens(x, r), up, r.ends))
    y = routing.combine_tokens(int8.grouped_linear_int8(h, down, r.ends), r)

All functions run on ``torch.cuda.current_stream()`` of their tensors' device,
take workspaces from PyTorch's caching allocator on it, do not synchronise,
give the same bits on every run, and raise ``ValueError`` for arguments that
they do not take. Calls with plain arguments are made by compiled code
(``csrc/expert_calls.cpp``); what it declines takes the path written out here,
to the same kernels.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Any

import torch
from torch.autograd import forward_ad

from . import _native_routing as nat
from ._native_calls import calls
from ._native_fp4 import raw_stream

_DTYPES = {torch.bfloat16: nat.DT_BF16, torch.float16: nat.DT_F16, torch.float32: nat.DT_F32}
_SCORING = {"softmax": nat.SOFTMAX, "sigmoid": nat.SIGMOID}
_GROUP_SCORE = {"max": nat.MAX, "top2": nat.TOP2}


@dataclass
class Routing:
    """Where the tokens of a batch go. ``weights`` fp32 and ``experts`` int32 (tokens, top_k), the best choice first, 0 and -1
    where a token has none; ``ends`` int32 (experts), the ends of the experts' groups in the order by expert, in which one
    expert's choices are in the order of their tokens; ``rows`` int32 (tokens, top_k), the place of each choice in it, or -1;
    ``source`` int32 (tokens * top_k), the choice ``token * top_k + slot`` at each place, or -1 past the last end. Every place
    below the last end belongs to one choice: a routing that is made otherwise has to keep to that, since the exchange neither
    adds up two choices at a place nor writes a place that has none."""

    weights: torch.Tensor
    experts: torch.Tensor
    ends: torch.Tensor
    rows: torch.Tensor
    source: torch.Tensor


def _dtype(t: torch.Tensor, what: str) -> int:
    dt = _DTYPES.get(t.dtype)
    if dt is None:
        raise ValueError(f"{what} supports bfloat16, float16 and float32 values, got {t.dtype}.")
    return dt


def _call(function: Any, device: torch.device, *args: Any) -> None:
    """A library call on the current stream of ``device``, with it current."""
    if torch.cuda.current_device() == device.index:
        nat.check(function(*args, raw_stream(device.index)))
    else:
        with torch.cuda.device(device):
            nat.check(function(*args, raw_stream(device.index)))


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x with contiguous rows that do not overlap (x itself where it has them)."""
    x = x.resolve_neg()
    if x.stride(1) != 1 or (x.stride(0) < x.shape[1] and x.shape[0] > 1):
        x = x.contiguous()
    return x


def _check_tangents(*tensors: torch.Tensor) -> None:
    if any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError("Routing has no forward-mode derivatives; detach the input's tangent.")


# ------------------------------------------------------------------------ routing
def _route(logits: torch.Tensor, config: nat.Config, bias: torch.Tensor | None, mask: torch.Tensor | None) -> tuple[torch.Tensor, ...]:
    x = _rows(logits)
    tokens, top_k = config.tokens, config.top_k
    weights = x.new_empty((tokens, top_k), dtype=torch.float32)
    experts, rows = (x.new_empty((tokens, top_k), dtype=torch.int32) for _ in range(2))
    ends, source = (x.new_empty(n, dtype=torch.int32) for n in (config.experts, tokens * top_k))
    lib, need = nat.load(), ctypes.c_size_t()
    ref = ctypes.byref(config)
    device = x.device
    with torch.cuda.device(device):
        nat.check(lib.piper_routing_workspace(ref, ctypes.byref(need)))
    ws = x.new_empty(need.value, dtype=torch.uint8) if need.value else None
    _call(lib.piper_routing_route, device, ref, x.data_ptr(), x.stride(0), _DTYPES[x.dtype], None if bias is None else bias.data_ptr(),
          None if mask is None else mask.data_ptr(), weights.data_ptr(), experts.data_ptr(), ends.data_ptr(), rows.data_ptr(),
          source.data_ptr(), None if ws is None else ws.data_ptr(), need.value)
    return weights, experts, ends, rows, source


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, config, bias, mask):
        out = _route(logits.detach(), config, bias, mask)
        ctx.save_for_backward(logits, out[1])
        ctx.config = config
        ctx.mark_non_differentiable(*out[1:])
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, *_):
        logits, experts = ctx.saved_tensors
        x = _rows(logits.detach())
        dlogits = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        _call(nat.load().piper_routing_route_grad, x.device, ctypes.byref(ctx.config), x.data_ptr(), x.stride(0), _DTYPES[x.dtype],
              experts.data_ptr(), grad.resolve_neg().contiguous().data_ptr(), dlogits.data_ptr())
        return dlogits, None, None, None


def route_tokens(logits: torch.Tensor, top_k: int, *, scoring: str = "softmax", bias: torch.Tensor | None = None, groups: int = 1,
                 top_groups: int | None = None, group_score: str = "max", renormalize: bool = True, scale: float = 1.0,
                 mask: torch.Tensor | None = None) -> Routing:
    """The ``top_k`` experts of each token from a router's ``logits`` (tokens, experts).

    ``scoring`` makes scores of the logits: ``"softmax"`` over the experts, or
    ``"sigmoid"`` of each. Choices go by score plus ``bias`` (fp32, one per
    expert) where there is one, in 64 bits where sums are near each other, else
    by the logits; the larger first, equal ones by index. With ``groups`` > 1
    neighbouring experts form that many equal groups, and choices come from the
    best ``top_groups`` of them: by their best choice (``group_score`` "max") or
    the sum of their two best ("top2"), equal ones by index. Weights are the
    scores without the bias, divided by their sum over the token's choices where
    ``renormalize``, times ``scale``. (A sum of sigmoids below 2**-100 counts as
    that. Softmax shares keep their proportions however small the scores are.)

    An expert with a logit or a bias of -infinity is closed: it is not chosen,
    and a token with fewer open experts than ``top_k`` has no choice in its last
    slots. A NaN comes after all numbers; softmax over a row with a NaN or
    +infinity gives the weight NaN. ``mask`` (bool, one per token): a token with
    False gets no expert. The weights are differentiable with respect to the
    logits; ``bias`` gets no gradient.
    """
    if scoring not in _SCORING:
        raise ValueError(f"Routing scores are softmax or sigmoid, got {scoring!r}.")
    if group_score not in _GROUP_SCORE:
        raise ValueError(f"A group's score is max or top2, got {group_score!r}.")
    if top_groups is None:
        top_groups = groups
    done = calls().route(logits, top_k, _SCORING[scoring], bias, groups, top_groups, _GROUP_SCORE[group_score], renormalize, scale, mask)
    if done is not None:
        return Routing(*done)
    if not logits.is_cuda:
        raise ValueError("Routing requires CUDA tensors.")
    if logits.ndim != 2:
        raise ValueError("route_tokens takes logits (tokens, experts).")
    _dtype(logits, "Routing")
    tokens, experts = logits.shape
    if bias is not None:
        if bias.dtype is not torch.float32 or bias.shape != (experts,) or bias.device != logits.device:
            raise ValueError("A routing bias is one float32 value per expert on the logits' device.")
        bias = bias.detach().resolve_neg().contiguous()
    if mask is not None:
        if mask.dtype is not torch.bool or mask.shape != (tokens,) or mask.device != logits.device:
            raise ValueError("A routing mask is one bool per token on the logits' device.")
        mask = mask.contiguous()
    limits = ((experts, nat.MAX_EXPERTS, "experts"), (top_k, nat.MAX_TOP_K, "experts for a token"), (groups, nat.MAX_GROUPS, "groups"))
    for value, most, what in limits:
        if not 1 <= value <= most:
            raise ValueError(f"Routing takes 1 to {most} {what}, got {value}.")
    config = nat.Config(tokens, experts, top_k, _SCORING[scoring], groups, top_groups, _GROUP_SCORE[group_score], bool(renormalize), scale)
    _check_tangents(logits)
    if logits.requires_grad and torch.is_grad_enabled():
        return Routing(*_Route.apply(logits, config, bias, mask))
    return Routing(*_route(logits.detach(), config, bias, mask))


# ----------------------------------------------------------------------- exchange
def _exchange(rows: torch.Tensor, ends: torch.Tensor, t: torch.Tensor, per_token: bool, what: str) -> nat.Exchange:
    """How ``t`` (a row per token, or per place) lies to a routing's rows, checked."""
    if not t.is_cuda:
        raise ValueError(f"{what} requires CUDA tensors.")
    dt = _dtype(t, what)
    for name, v in (("rows", rows), ("ends", ends)):
        if v.dtype is not torch.int32 or not v.is_contiguous() or v.device != t.device:
            raise ValueError(f"A routing's {name} are contiguous int32 on the device of the tokens.")
    if rows.ndim != 2 or ends.ndim != 1 or ends.shape[0] == 0:
        raise ValueError("A routing has rows (tokens, top_k) and ends (experts).")
    tokens, top_k = rows.shape
    want = tokens if per_token else tokens * top_k
    if t.ndim != 2 or t.shape[0] != want:
        raise ValueError(f"{what} takes {want} rows, got {tuple(t.shape)}.")
    if t.shape[1] == 0:
        raise ValueError(f"{what} requires rows with values.")
    return nat.Exchange(tokens, top_k, t.shape[1], dt, rows.data_ptr(), ends.data_ptr() + 4 * (ends.shape[0] - 1))


def _dispatch(x: torch.Tensor, rows: torch.Tensor, ends: torch.Tensor) -> torch.Tensor:
    e = _exchange(rows, ends, x, True, "dispatch_tokens")
    x2 = _rows(x.detach())
    out = x.new_empty((rows.numel(), x.shape[1]))
    _call(nat.load().piper_routing_dispatch, x.device, ctypes.byref(e), x2.data_ptr(), x2.stride(0), out.data_ptr())
    return out


def _combine(y: torch.Tensor, rows: torch.Tensor, ends: torch.Tensor, weights: torch.Tensor | None, what: str) -> torch.Tensor:
    e = _exchange(rows, ends, y, False, what)
    y2 = _rows(y.detach())
    out = y.new_empty((rows.shape[0], y.shape[1]))
    _call(nat.load().piper_routing_combine, y.device, ctypes.byref(e), y2.data_ptr(), y2.stride(0),
          None if weights is None else weights.data_ptr(), out.data_ptr())
    return out


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, rows, ends):
        ctx.save_for_backward(rows, ends)
        return _dispatch(x, rows, ends)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return _combine(grad, *ctx.saved_tensors, None, "dispatch_tokens' gradient"), None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, rows, ends):
        ctx.save_for_backward(y, weights, rows, ends)
        return _combine(y, rows, ends, weights, "combine_tokens")

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        y, weights, rows, ends = ctx.saved_tensors
        e = _exchange(rows, ends, y, False, "combine_tokens' gradient")
        y2, g2 = _rows(y.detach()), _rows(grad)
        dy = torch.empty(y.shape, dtype=y.dtype, device=y.device)
        dweights = torch.empty(weights.shape, dtype=torch.float32, device=y.device)
        _call(nat.load().piper_routing_combine_grad, y.device, ctypes.byref(e), y2.data_ptr(), y2.stride(0), weights.data_ptr(),
              g2.data_ptr(), g2.stride(0), dy.data_ptr(), dweights.data_ptr())
        return dy, dweights, None, None


def dispatch_tokens(x: torch.Tensor, routing: Routing) -> torch.Tensor:
    """``x`` (tokens, hidden) copied to the places of its choices: (tokens * top_k, hidden), sorted by expert, zeros past the
    last end. Its gradient adds the copies' up, in fp32 in the order of the slots, rounded once."""
    rows, ends = routing.rows, routing.ends
    done = calls().dispatch(x, rows, ends)
    if done is not None:
        return done
    _check_tangents(x)
    if x.requires_grad and torch.is_grad_enabled():
        return _Dispatch.apply(x, rows, ends)
    return _dispatch(x, rows, ends)


def combine_tokens(y: torch.Tensor, routing: Routing) -> torch.Tensor:
    """The experts' rows ``y`` (tokens * top_k, hidden) added up for each token by its weights: (tokens, hidden), in fp32 in the
    order of the slots, rounded once. A token without a choice gets zeros. Differentiable with respect to ``y`` and to the
    routing's weights."""
    rows, ends, weights = routing.rows, routing.ends, routing.weights
    done = calls().combine(y, weights, rows, ends)
    if done is not None:
        return done
    if weights.dtype is not torch.float32 or weights.shape != rows.shape or weights.device != rows.device:
        raise ValueError("A routing's weights are float32, one for each choice.")
    weights = weights.resolve_neg().contiguous()
    _check_tangents(y, weights)
    if (y.requires_grad or weights.requires_grad) and torch.is_grad_enabled():
        return _Combine.apply(y, weights, rows, ends)
    return _combine(y, rows, ends, weights, "combine_tokens")
