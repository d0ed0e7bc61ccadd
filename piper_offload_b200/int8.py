"""8-bit integer products with the INT8 weights that the merges change, and the products' gradients.

The merges change packed weights in place; these functions multiply with them,
on sm_100a kernels of ``libpiper_int8.so``:

* :func:`linear_int8`: tokens times a weight, the tokens quantised to 8 bits on
  the way;
* :func:`grouped_linear_int8`: the same with one weight per expert, the tokens
  sorted by expert and the ends of their groups on the device (as
  :func:`~.routing.route_tokens` and :func:`~.routing.dispatch_tokens` make them);
* :func:`linear_int8_grad_input`, :func:`grouped_linear_int8_grad_input`: the
  gradients with respect to the tokens. The two products are differentiable:
  they use these when their input requires a gradient. Weights are constants,
  the gradients are not differentiable themselves, and inputs with a
  forward-mode tangent are refused.

Weights (:mod:`~.weights`, or tensors of the libraries with the same
attributes): ``Int8Weight`` with a scale, and a zero point where there is one,
for each row or for the whole weight; ``Int8Experts``, a stack of them with a
scale for each row; ``Bnb8Weight`` (LLM.int8); ``QuantoWeight`` of qint8 with a
scale for each row or one for all. Groups of columns, scales for columns and
``act_pre_scale`` are refused. Tokens are quantised to 8 bits for all of them,
also where the weight's library would multiply by dequantised weights.

Definitions. A weight's value is ``(code - zero) * scale`` (LLM.int8: ``code *
SCB / 127``). A token with the largest magnitude ``a`` is held as the codes
``rint(127 * x / a)``, ties to even, and the scale ``a / 127``; the product is
the whole-number sum of codes times both scales, ``(sum * token's) * row's`` in
fp32, rounded once to the type of the token. A token that holds an infinity or
a NaN gives a row of NaN and touches no other. The gradient goes straight
through the quantisation of the tokens: ``dx = (dy * scale) @ (codes - zero)``
with fp32 sums, in which ``dy * scale`` is rounded to 11 bits for bf16 and fp16
gradients: that adds 1 % to the error that the rounding of a bf16 result makes,
and 40 % to an fp16 one's. For fp32 gradients it has 22 bits, at twice the
products; a caller who wants them passes ``dy.float()`` (or ``x.float()`` to a
product that is differentiated).

All functions run on ``torch.cuda.current_stream()`` of their tensors' device,
take workspaces from PyTorch's caching allocator on it, do not synchronise,
and raise ``ValueError`` for arguments that they do not take. Calls with plain
arguments are made by compiled code (``csrc/expert_calls.cpp``); what it
declines takes the path written out here, to the same kernels. Quanto weights
always do: 18 us of host time a call, 5 for the others.
"""

from __future__ import annotations

import ctypes
from typing import Any

import torch
from torch.autograd import forward_ad

from . import _native_int8 as nat
from . import kernels as K
from ._native_calls import calls
from ._native_fp4 import raw_stream
from .adapters import Bnb8Adapter, Int8Adapter, QuantoAdapter
from .weights import Bnb8Weight, Int8Experts, Int8Weight, QuantoWeight

_DTYPES = {torch.bfloat16: nat.DT_BF16, torch.float16: nat.DT_F16, torch.float32: nat.DT_F32}


def _dtype(t: torch.Tensor, what: str) -> int:
    dt = _DTYPES.get(t.dtype)
    if dt is None:
        raise ValueError(f"INT8 {what} supports bfloat16, float16 and float32 values, got {t.dtype}.")
    return dt


class _Frozen:
    """A weight's tensors as they are now, checked: what one product and its backward pass work with. A tensor that is put
    in another's place in between changes nothing."""

    __slots__ = ("codes", "scale", "zero", "matrix", "_versions")

    def __init__(self, w: Any, dims: int):
        zero, over_127, per_row = None, False, True
        if Bnb8Adapter.matches(w):
            codes, scale, over_127 = w.CB, w.SCB, True
        elif QuantoAdapter.matches(w):
            codes, scale = w._data, w._scale
            if codes.dtype is torch.int8 and codes.ndim == 2:
                layout = K.quanto_scale_axis(w.axis, scale, *codes.shape)
                if layout == "column":
                    raise ValueError("INT8 products do not take scales for columns.")
                per_row = layout == "row"
        elif Int8Adapter.matches(w):
            codes, scale, zero = w.qdata, w.scale, getattr(w, "zero_point", None)
            if getattr(w, "act_pre_scale", None) is not None:
                raise ValueError("INT8 products do not take act_pre_scale; scale the tokens before the product.")
            block = tuple(w.block_size)[-2:]
            per_row = len(block) == 2 and block[0] == 1
            if len(block) != 2 or block[1] != codes.shape[-1] or not (per_row or block[0] == codes.shape[-2]):
                raise ValueError(f"INT8 products take a scale for each row or one for all, got blocks of {tuple(w.block_size)}.")
        else:
            raise ValueError(f"INT8 products take INT8 weights, got {type(w).__name__}.")
        if codes.ndim != dims:
            raise ValueError("linear_int8 takes one weight, grouped_linear_int8 a stack of experts.")
        if not codes.is_cuda:
            raise ValueError("INT8 operators require CUDA tensors.")
        if codes.dtype is not torch.int8:
            raise ValueError(f"INT8 operators expect int8 codes, got {codes.dtype}.")
        batch, (rows, cols) = (codes.shape[0] if dims == 3 else 1), codes.shape[-2:]
        if batch == 0 or rows == 0 or cols == 0:
            raise ValueError("INT8 operators require non-empty weights.")
        if dims == 3 and not per_row:
            raise ValueError("INT8 experts have a scale for each row.")
        values, scale = batch * rows if per_row else 1, scale.resolve_neg()
        if scale.dtype not in _DTYPES:
            raise ValueError(f"INT8 scales are bfloat16, float16 or float32, got {scale.dtype}.")
        if scale.numel() != values:
            raise ValueError(f"INT8 scale shape {tuple(scale.shape)} does not match its weight's {tuple(codes.shape)}.")
        if zero is not None and (zero.dtype is not torch.int8 or zero.numel() != values):
            raise ValueError("INT8 zero points are int8 values, one for each scale.")
        for t in (codes, scale, zero):
            if t is not None and (t.device != codes.device or not t.is_contiguous()):
                raise ValueError("INT8 operators require contiguous tensors on one CUDA device.")
        self.codes, self.scale, self.zero = codes, scale, zero
        self.matrix = nat.Matrix(codes.data_ptr(), scale.data_ptr(), None if zero is None else zero.data_ptr(), batch, rows, cols,
                                 _DTYPES[scale.dtype], per_row, over_127)
        self._versions = None

    def mark(self) -> None:
        self._versions = [(t, t._version) for t in (self.codes, self.scale, self.zero) if t is not None and not t.is_inference()]

    def check(self) -> None:
        if any(t._version != version for t, version in self._versions):
            raise RuntimeError("a tensor of an INT8 weight has been modified by an inplace operation since its product, "
                               "whose gradient needs it as it was.")


def _on(device: torch.device, function: Any, *args: Any) -> None:
    """A library call with ``device`` current: plans and launches alike depend on it."""
    if torch.cuda.current_device() == device.index:
        nat.check(function(*args))
    else:
        with torch.cuda.device(device):
            nat.check(function(*args))


def _workspace(query: Any, device: torch.device, *args: Any) -> torch.Tensor | None:
    need = ctypes.c_size_t()
    _on(device, query, *args, ctypes.byref(need))
    return torch.empty(need.value, dtype=torch.uint8, device=device) if need.value else None


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x as a matrix whose rows are contiguous and do not overlap (a view where it is one)."""
    x = x.resolve_neg()
    if x.ndim != 2:
        x = x.reshape(-1, x.shape[-1])
    if x.stride(1) != 1 or (x.stride(0) < x.shape[1] and x.shape[0] > 1):
        x = x.contiguous()
    return x


def _check_tangents(*tensors: torch.Tensor) -> None:
    if any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError("INT8 operators have no forward-mode derivatives; detach the input's tangent.")


def _check_ends(ends: torch.Tensor, w: _Frozen) -> None:
    if ends.dtype is not torch.int32 or ends.ndim != 1 or ends.shape[0] != w.matrix.batch or not ends.is_contiguous():
        raise ValueError("Group ends are one contiguous int32 vector with an entry per expert.")
    if ends.device != w.codes.device:
        raise ValueError("INT8 operators require all tensors on one CUDA device.")


def _run(x: torch.Tensor, w: _Frozen, ends: torch.Tensor | None, grad: bool) -> torch.Tensor:
    """The product of tokens, or the gradient from that of its result."""
    m, device = w.matrix, w.codes.device
    into, out = (m.rows, m.cols) if grad else (m.cols, m.rows)
    if x.device != device:
        raise ValueError("INT8 operators require all tensors on one CUDA device.")
    dt = _dtype(x, "gradient" if grad else "product")
    if x.ndim < 1 or x.shape[-1] != into:
        raise ValueError(f"INT8 gradient: the output's gradient has {tuple(x.shape)}, the weight {into} rows." if grad else
                         f"INT8 product: the input has {tuple(x.shape)}, the weight {into} columns.")
    if ends is not None:
        _check_ends(ends, w)
    x2 = _rows(x.detach())
    tokens = x2.shape[0]
    y = x.new_empty((*x.shape[:-1], out))
    lib, ref = nat.load(), ctypes.byref(m)
    if tokens == 0:
        return y
    if grad:
        ws = _workspace(lib.piper_int8_grad_input_workspace, device, ref, tokens, dt)
    else:
        ws = _workspace(lib.piper_int8_linear_workspace, device, ref, tokens, ends is not None)
    _on(device, lib.piper_int8_grad_input if grad else lib.piper_int8_linear, ref, x2.data_ptr(), x2.stride(0), tokens,
        None if ends is None else ends.data_ptr(), y.data_ptr(), dt, *((None, 0) if ws is None else (ws.data_ptr(), ws.numel())),
        raw_stream(device.index))
    return y


class _Product(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, ends):
        ctx.save_for_backward(ends)
        weight.mark()
        ctx.weight = weight
        return _run(x, weight, ends, False)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (ends,) = ctx.saved_tensors
        ctx.weight.check()
        return _run(grad, ctx.weight, ends, True), None, None


def _product(x: torch.Tensor, weight: Any, ends: torch.Tensor | None) -> torch.Tensor:
    done = calls().int8(x, weight, ends, False)
    if done is not None:
        return done
    w = _Frozen(weight, 2 if ends is None else 3)
    _check_tangents(x)
    if x.requires_grad and torch.is_grad_enabled():
        return _Product.apply(x, w, ends)
    return _run(x, w, ends, False)


def _grad_input(grad: torch.Tensor, weight: Any, ends: torch.Tensor | None) -> torch.Tensor:
    done = calls().int8(grad, weight, ends, True)
    if done is not None:
        return done
    _check_tangents(grad)
    return _run(grad, _Frozen(weight, 2 if ends is None else 3), ends, True)


def linear_int8(x: torch.Tensor, weight: Int8Weight | Bnb8Weight | QuantoWeight) -> torch.Tensor:
    """``quantised(x) @ weight.T`` for ``x`` (..., cols); the result is (..., rows) in the type of ``x``.

    Differentiable with respect to ``x`` (straight through its quantisation);
    the weight is constant. Between the two passes its tensors may be replaced,
    and an operation of torch that changes them raises. A merge into them is not
    noticed: the gradient is the merged one's.
    """
    return _product(x, weight, None)


def grouped_linear_int8(x: torch.Tensor, experts: Int8Experts, group_ends: torch.Tensor) -> torch.Tensor:
    """:func:`linear_int8` with a weight per expert over rows sorted by expert.

    ``x`` is (tokens, cols); expert ``e`` has the rows ``group_ends[e - 1]`` to
    ``group_ends[e]`` (int32 on the device, non-decreasing, not read by the
    host). Experts may have no rows; rows past the last end come out as zeros.
    An end below one before it counts as that one, one past the tokens as theirs.
    """
    if x.ndim != 2:
        raise ValueError("grouped_linear_int8 takes a stack of experts and rank-two tokens.")
    return _product(x, experts, group_ends)


def linear_int8_grad_input(grad: torch.Tensor, weight: Int8Weight | Bnb8Weight | QuantoWeight) -> torch.Tensor:
    """``grad @ values(weight)`` for ``grad`` (..., rows): :func:`linear_int8`'s gradient, in the type of ``grad``."""
    return _grad_input(grad, weight, None)


def grouped_linear_int8_grad_input(grad: torch.Tensor, experts: Int8Experts, group_ends: torch.Tensor) -> torch.Tensor:
    """:func:`grouped_linear_int8`'s gradient with respect to its tokens; rows past the last end get zeros."""
    if grad.ndim != 2:
        raise ValueError("grouped_linear_int8_grad_input takes a stack of experts and a rank-two gradient.")
    return _grad_input(grad, experts, group_ends)
