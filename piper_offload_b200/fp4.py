"""4-bit floating-point operators around the merge: make FP4 weights, use them, differentiate through them.

The merges change packed weights in place; these functions make such weights
from dense ones and multiply with them, in the layouts the merges read and
write (:class:`~.weights.MXWeight` with e2m1 elements, :class:`~.weights.NVFP4Weight`,
and their stacks of experts), on sm_100a kernels of ``libpiper_fp4.so``:

* :func:`quantize_mxfp4`, :func:`quantize_nvfp4`, :func:`dequantize_fp4`;
* :func:`linear_fp4`: tokens times a weight, the tokens quantised on the way;
* :func:`grouped_linear_fp4`: the same with one weight per expert, the tokens
  sorted by expert and the ends of their groups on the device;
* :func:`linear_fp4_grad_input`, :func:`grouped_linear_fp4_grad_input`: the
  gradients with respect to the tokens. The two products are differentiable:
  they use these when their input requires a gradient. Weights and second-level
  scales are constants, the gradients are not differentiable themselves, and
  inputs with a forward-mode tangent are refused.

Definitions. A block of a row (32 values in MXFP4, 16 in NVFP4) with the
largest magnitude ``a`` is stored as ``e2m1(clamp(x / s, -6, 6)) * s``, nearest
with ties to even. MXFP4: ``s`` is a power of two that ``scaling_mode`` derives
from ``a``. NVFP4: ``s = e4m3(clamp(a / 6 / g, 2**-6, 448)) * g``, where the
second-level scale ``g`` is 1, given, or ``max(max|x| / 2688, 2**-23)`` over
the matrix's finite values. A block that holds a NaN reads back as NaN; an
infinity saturates its block's scale.
Products are over these values, summed in fp32 and rounded once to the type
of the tokens. Second-level scales multiply the sum, so it is the sum before
them that has to fit fp32.

All functions run on ``torch.cuda.current_stream()`` of their tensors' device,
take workspaces from PyTorch's caching allocator on it, do not synchronise,
and raise ``ValueError`` for arguments that they do not take. Calls with plain
arguments are made by compiled code (``csrc/fp4_calls.cpp``); what it declines
takes the path written out here, to the same kernels.
"""

from __future__ import annotations

import ctypes
from typing import Any

import torch
from torch.autograd import forward_ad

from . import _native_fp4 as nat
from . import kernels as K
from .adapters import mx_scaling_mode_id
from .weights import MXActQuantKwargs, MXExperts, MXScalingMode, MXWeight, NVFP4Experts, NVFP4Weight

_DTYPES = {torch.bfloat16: nat.DT_BF16, torch.float32: nat.DT_F32}
_FP4 = K._FP4_DTYPE
_E8M0 = K._E8M0_DTYPE


def _dtype(t: torch.Tensor, what: str) -> int:
    dt = _DTYPES.get(t.dtype)
    if dt is None:
        raise ValueError(f"FP4 {what} supports bfloat16 and float32 values, got {t.dtype}.")
    return dt


def _matrix(w: Any) -> tuple[nat.Matrix, int, torch.Tensor]:
    """(descriptor, MX scaling mode of activations, codes) of a packed weight or stack, checked."""
    q, s = w.qdata, w.scale
    if not q.is_cuda:
        raise ValueError("FP4 operators require CUDA tensors.")
    if q.dtype is not torch.uint8:
        raise ValueError(f"FP4 operators expect packed uint8 codes, got {q.dtype}.")
    shape, scale_shape = q.shape, s.shape
    if len(shape) == 2:
        batch, (rows, cols) = 1, shape
    elif len(shape) == 3:
        batch, rows, cols = shape
        if len(scale_shape) == 3 and scale_shape[0] != batch:
            raise ValueError(f"FP4 scale shape {tuple(scale_shape)} does not match its layout.")
    if len(shape) not in (2, 3) or len(scale_shape) != len(shape):
        raise ValueError("FP4 operators expect rank-two weights, or rank-three stacks of experts.")
    cols *= 2
    if not q.is_contiguous() or not s.is_contiguous():
        raise ValueError("FP4 operators require contiguous codes and scales.")
    if s.device != q.device:
        raise ValueError("FP4 operators require all tensors on one CUDA device.")
    if batch == 0 or rows == 0 or cols == 0:
        raise ValueError("FP4 operators require non-empty weights.")
    swizzled = bool(w.is_swizzled_scales)
    second = None
    elem = getattr(w, "elem_dtype", None)
    if elem is not None:
        if elem is not _FP4 or _FP4 is None:
            raise ValueError(f"FP4 operators support MX weights with e2m1 elements, got {elem}.")
        if w.block_size != 32 or cols % 32:
            raise ValueError("MXFP4 weights have blocks of 32 and columns divisible by 32.")
        if s.dtype is not torch.uint8 and s.dtype is not _E8M0:
            raise ValueError(f"MXFP4 weights have E8M0 scales, got {s.dtype}.")
        expected = K.mx_expected_scale_shape(rows, cols, swizzled=swizzled)
        mode = mx_scaling_mode_id(w)
        if mode is None:
            raise ValueError("MXFP4 activations support FLOOR, RCEIL, CEIL and EVEN scale rounding.")
        fmt = nat.FMT_MX
    else:
        if w.block_size != 16 or cols % 16:
            raise ValueError("NVFP4 weights have blocks of 16 and columns divisible by 16.")
        if s.dtype is not torch.float8_e4m3fn:
            raise ValueError(f"NVFP4 weights have E4M3FN scales, got {s.dtype}.")
        expected = K.nvfp4_expected_scale_shape(rows, cols, swizzled=swizzled)
        second = w.per_tensor_scale
        if second is not None and (second.dtype is not torch.float32 or second.numel() != batch
                                   or second.device != q.device or not second.is_contiguous()):
            raise ValueError("NVFP4 second-level scales are one contiguous float32 value per matrix on its device.")
        fmt, mode = nat.FMT_NV, 0
    if scale_shape[-2:] != expected:
        raise ValueError(f"FP4 scale shape {tuple(scale_shape)} does not match its layout.")
    m = nat.Matrix(q.data_ptr(), s.data_ptr(), None if second is None else second.data_ptr(), batch, rows, cols, fmt,
                   swizzled)
    return m, mode, q


def _on(device: torch.device, function: Any, *args: Any) -> None:
    """A library call with ``device`` current: plans and launches alike depend on it."""
    if torch.cuda.current_device() == device.index:
        nat.check(function(*args))
    else:
        with torch.cuda.device(device):
            nat.check(function(*args))


def _call(function: Any, device: torch.device, *args: Any) -> None:
    """A library call on the current stream of ``device``."""
    _on(device, function, *args, nat.raw_stream(device.index))


def _workspace(query: Any, device: torch.device, *args: Any) -> torch.Tensor | None:
    need = ctypes.c_size_t()
    _on(device, query, *args, ctypes.byref(need))
    return torch.empty(need.value, dtype=torch.uint8, device=device) if need.value else None


def _span(workspace: torch.Tensor | None) -> tuple[int | None, int]:
    return (None, 0) if workspace is None else (workspace.data_ptr(), workspace.numel())


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x as a matrix whose rows are contiguous and do not overlap (a view where it is one)."""
    if x.ndim != 2:
        x = x.reshape(-1, x.shape[-1])
    if x.stride(1) != 1 or (x.stride(0) < x.shape[1] and x.shape[0] > 1):
        x = x.contiguous()
    return x


# ------------------------------------------------------------------ quantisation
def _quantize(x: torch.Tensor, fmt: int, mode: int, swizzled: bool, second: torch.Tensor | None,
              second_mode: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    done = nat.calls().quantize(x, fmt, mode, swizzled, second_mode)
    if done is not None:
        return done
    block = 32 if fmt == nat.FMT_MX else 16
    if not x.is_cuda:
        raise ValueError("FP4 quantisation requires CUDA tensors.")
    dt = _dtype(x, "quantisation")
    if x.ndim not in (2, 3):
        raise ValueError("FP4 quantisation expects a matrix, or a stack of them.")
    rows, cols = x.shape[-2:]
    if x.numel() == 0:
        raise ValueError("FP4 quantisation requires non-empty tensors.")
    if cols % block:
        raise ValueError(f"{'MXFP4' if fmt == nat.FMT_MX else 'NVFP4'} quantisation requires columns divisible by {block}.")
    x2 = _rows(x.detach())
    lead = x.shape[:-2]
    shape = (K.mx_expected_scale_shape if fmt == nat.FMT_MX else K.nvfp4_expected_scale_shape)(rows, cols, swizzled=swizzled)
    codes = x.new_empty((*lead, rows, cols // 2), dtype=torch.uint8)
    scale = x.new_empty((*lead, *shape), dtype=torch.uint8 if fmt == nat.FMT_MX else torch.float8_e4m3fn)
    if second_mode == nat.SECOND_COMPUTE:
        second = x.new_empty(lead[0] if lead else 1, dtype=torch.float32)
    m = nat.Matrix(codes.data_ptr(), scale.data_ptr(), None if second is None else second.data_ptr(),
                   lead[0] if lead else 1, rows, cols, fmt, swizzled)
    maxima = None
    if second_mode == nat.SECOND_COMPUTE and rows * cols > nat.SMALL_MATRIX:
        maxima = x.new_empty(m.batch, dtype=torch.int32)
    _call(nat.load().piper_fp4_quantize, x.device, ctypes.byref(m), x2.data_ptr(), x2.stride(0), dt, mode, second_mode,
          None if maxima is None else maxima.data_ptr())
    return codes, scale, second


def quantize_mxfp4(x: torch.Tensor, *, scaling_mode: str | int = "floor", swizzled: bool = False) -> MXWeight | MXExperts:
    """``x`` (rows, cols), or a stack (experts, rows, cols), as MXFP4.

    ``scaling_mode`` is kept with the result: its tokens are quantised the same way.
    """
    name = {v: k for k, v in K._MX_SCALING_MODES.items()}.get(scaling_mode, scaling_mode)
    if name not in K._MX_SCALING_MODES:
        raise ValueError(f"Unsupported MX scaling mode {scaling_mode!r}.")
    if _FP4 is None:
        raise ValueError("MXFP4 weights need torch.float4_e2m1fn_x2.")
    codes, scale, _ = _quantize(x, nat.FMT_MX, K._MX_SCALING_MODES[name], swizzled, None, nat.SECOND_NONE)
    kind = MXExperts if x.ndim == 3 else MXWeight
    return kind(codes, scale, _FP4, orig_dtype=x.dtype, is_swizzled_scales=swizzled,
                act_quant_kwargs=MXActQuantKwargs(MXScalingMode(name)))


def quantize_nvfp4(x: torch.Tensor, *, two_level: bool = True, per_tensor_scale: torch.Tensor | None = None,
                   swizzled: bool = False) -> NVFP4Weight | NVFP4Experts:
    """``x`` (rows, cols), or a stack (experts, rows, cols), as NVFP4.

    With ``two_level`` each matrix gets a second-level scale: ``per_tensor_scale``
    (fp32, one per matrix) where given, else one computed from its largest value.
    """
    batch = x.shape[0] if x.ndim == 3 else 1
    second, second_mode = None, nat.SECOND_NONE
    if per_tensor_scale is not None:
        if not two_level:
            raise ValueError("NVFP4 quantisation without a second level takes no per_tensor_scale.")
        if (per_tensor_scale.dtype is not torch.float32 or per_tensor_scale.numel() != batch
                or per_tensor_scale.device != x.device):
            raise ValueError("NVFP4 second-level scales are one float32 value per matrix on its device.")
        second, second_mode = per_tensor_scale.detach().reshape(batch).contiguous(), nat.SECOND_GIVEN
    elif two_level:
        second_mode = nat.SECOND_COMPUTE
    codes, scale, second = _quantize(x, nat.FMT_NV, 0, swizzled, second, second_mode)
    kind = NVFP4Experts if x.ndim == 3 else NVFP4Weight
    return kind(codes, scale, second, orig_dtype=x.dtype, is_swizzled_scales=swizzled)


def dequantize_fp4(weight: Any, dtype: torch.dtype | None = None) -> torch.Tensor:
    """The values of a packed weight or stack, rounded once to ``dtype`` (default: the weight's original type)."""
    if getattr(weight, "qdata", None) is None:
        raise ValueError(f"FP4 operators take MXFP4 and NVFP4 weights, got {type(weight).__name__}.")
    done = nat.calls().dequantize(weight, weight.qdata.ndim, dtype)
    if done is not None:
        return done
    m, _, q = _matrix(weight)
    y = q.new_empty((*q.shape[:-1], m.cols), dtype=dtype or weight.orig_dtype)
    _call(nat.load().piper_fp4_dequantize, q.device, ctypes.byref(m), y.data_ptr(), _dtype(y, "dequantisation"))
    return y


# ---------------------------------------------------------------------- products
def _check_kind(weight: Any, dims: int, message: str) -> None:
    if getattr(weight, "qdata", None) is None:
        raise ValueError(f"FP4 operators take MXFP4 and NVFP4 weights, got {type(weight).__name__}.")
    if weight.qdata.ndim != dims:
        raise ValueError(message)


def _check_tangents(*tensors: torch.Tensor | None) -> None:
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError("FP4 operators have no forward-mode derivatives; detach the input's tangent.")


def _check_ends(ends: torch.Tensor, batch: int, device: torch.device) -> None:
    if ends.dtype is not torch.int32 or ends.ndim != 1 or ends.shape[0] != batch or not ends.is_contiguous():
        raise ValueError("Group ends are one contiguous int32 vector with an entry per expert.")
    if ends.device != device:
        raise ValueError("FP4 operators require all tensors on one CUDA device.")


def _linear(x: torch.Tensor, weight: Any, ends: torch.Tensor | None, act_scale: torch.Tensor | None) -> torch.Tensor:
    done = nat.calls().linear(x, weight, ends, act_scale)
    if done is not None:
        return done
    _check_tangents(x, act_scale)
    m, mode, q = _matrix(weight)
    device = q.device
    if x.device != device:
        raise ValueError("FP4 operators require all tensors on one CUDA device.")
    dt = _dtype(x, "product")
    if x.ndim < 1 or x.shape[-1] != m.cols:
        raise ValueError(f"FP4 product: the input has {tuple(x.shape)}, the weight {m.cols} columns.")
    if act_scale is not None:
        if m.format != nat.FMT_NV:
            raise ValueError("MXFP4 activations have no second-level scale.")
        if act_scale.dtype is not torch.float32 or act_scale.numel() != 1 or act_scale.device != device:
            raise ValueError("The activations' second-level scale is one float32 value on their device.")
    x2 = _rows(x)
    tokens = x2.shape[0]
    y = x.new_empty((tokens, m.rows) if x2 is x else (*x.shape[:-1], m.rows))
    if tokens == 0:
        return y
    lib, ref = nat.load(), ctypes.byref(m)
    ws = _workspace(lib.piper_fp4_linear_workspace, device, ref, tokens)
    _call(lib.piper_fp4_linear, device, ref, x2.data_ptr(), x2.stride(0), tokens, None if ends is None else ends.data_ptr(),
          None if act_scale is None else act_scale.data_ptr(), mode, y.data_ptr(), dt, *_span(ws))
    return y


def _grad_input(grad: torch.Tensor, weight: Any, ends: torch.Tensor | None) -> torch.Tensor:
    done = nat.calls().grad_input(grad, weight, ends)
    if done is not None:
        return done
    _check_tangents(grad)
    m, _, q = _matrix(weight)
    device = q.device
    if grad.device != device:
        raise ValueError("FP4 operators require all tensors on one CUDA device.")
    dt = _dtype(grad, "gradient")
    if grad.ndim < 1 or grad.shape[-1] != m.rows:
        raise ValueError(f"FP4 gradient: the output's gradient has {tuple(grad.shape)}, the weight {m.rows} rows.")
    g2 = _rows(grad)
    tokens = g2.shape[0]
    dx = grad.new_empty((tokens, m.cols) if g2 is grad else (*grad.shape[:-1], m.cols))
    if tokens == 0:
        return dx
    lib, ref = nat.load(), ctypes.byref(m)
    ws = None
    if dt != nat.DT_BF16 or g2.data_ptr() % 16 or g2.stride(0) % 8:  # bf16 rows that bulk copies can read need none
        ws = _workspace(lib.piper_fp4_grad_input_workspace, device, ref, g2.data_ptr(), g2.stride(0), tokens, dt)
    _call(lib.piper_fp4_grad_input, device, ref, g2.data_ptr(), g2.stride(0), tokens, None if ends is None else ends.data_ptr(),
          dx.data_ptr(), dt, *_span(ws))
    return dx


class _Frozen:
    """The parts of a weight as its product found them, for the backward pass: a part that is put in another's place
    in between changes nothing. Not saved tensors, since hooks on those would move a weight that stays in use."""

    def __init__(self, weight: Any):
        for name in ("qdata", "scale", "per_tensor_scale", "block_size", "elem_dtype", "is_swizzled_scales", "act_quant_kwargs"):
            if hasattr(weight, name):
                setattr(self, name, getattr(weight, name))
        tensors = (self.qdata, self.scale, getattr(self, "per_tensor_scale", None))
        self._versions = [(t, t._version) for t in tensors if t is not None and not t.is_inference()]

    def check(self) -> None:
        if any(t._version != version for t, version in self._versions):
            raise RuntimeError("a tensor of an FP4 weight has been modified by an inplace operation since its product, "
                               "whose gradient needs it as it was.")


class _Product(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, ends, act_scale):
        ctx.save_for_backward(ends)
        ctx.weight = _Frozen(weight)
        return _linear(x, weight, ends, act_scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (ends,) = ctx.saved_tensors
        ctx.weight.check()
        return _grad_input(grad, ctx.weight, ends), None, None, None


def _product(x: torch.Tensor, weight: Any, ends: torch.Tensor | None, act_scale: torch.Tensor | None) -> torch.Tensor:
    if x.requires_grad and torch.is_grad_enabled():
        _check_tangents(x, act_scale)
        return _Product.apply(x, weight, ends, act_scale)
    return _linear(x, weight, ends, act_scale)


def linear_fp4(x: torch.Tensor, weight: MXWeight | NVFP4Weight, *,
               act_per_tensor_scale: torch.Tensor | None = None) -> torch.Tensor:
    """``quantised(x) @ weight.T`` for ``x`` (..., cols); the result is (..., rows) in the type of ``x``.

    ``x`` is quantised in the weight's format: MXFP4 with the weight's
    ``act_quant_kwargs.scaling_mode``, NVFP4 with the second-level scale
    ``act_per_tensor_scale`` where one is given. Differentiable with respect to
    ``x`` (straight through its quantisation); the weight is constant. Between the
    two passes its tensors may be replaced, and an operation of torch that
    changes them raises. A merge into them is not noticed: the gradient is the
    merged one's.
    """
    _check_kind(weight, 2, "linear_fp4 takes one weight; grouped_linear_fp4 takes a stack of experts.")
    return _product(x, weight, None, act_per_tensor_scale)


def grouped_linear_fp4(x: torch.Tensor, experts: MXExperts | NVFP4Experts, group_ends: torch.Tensor, *,
                       act_per_tensor_scale: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`linear_fp4` with a weight per expert over rows sorted by expert.

    ``x`` is (tokens, cols); expert ``e`` has the rows ``group_ends[e - 1]`` to
    ``group_ends[e]`` (int32 on the device, non-decreasing, not read by the
    host). Experts may have no rows; rows past the last end come out as zeros.
    An end below one before it counts as that one, one past the tokens as theirs.
    """
    _check_kind(experts, 3, "grouped_linear_fp4 takes a stack of experts and rank-two tokens.")
    if x.ndim != 2:
        raise ValueError("grouped_linear_fp4 takes a stack of experts and rank-two tokens.")
    _check_ends(group_ends, experts.qdata.shape[0], experts.qdata.device)
    return _product(x, experts, group_ends, act_per_tensor_scale)


def linear_fp4_grad_input(grad: torch.Tensor, weight: MXWeight | NVFP4Weight) -> torch.Tensor:
    """``grad @ dequantised(weight)`` for ``grad`` (..., rows): :func:`linear_fp4`'s gradient, in the type of ``grad``."""
    _check_kind(weight, 2, "linear_fp4_grad_input takes one weight; grouped_linear_fp4_grad_input takes a stack of experts.")
    return _grad_input(grad, weight, None)


def grouped_linear_fp4_grad_input(grad: torch.Tensor, experts: MXExperts | NVFP4Experts,
                                  group_ends: torch.Tensor) -> torch.Tensor:
    """:func:`grouped_linear_fp4`'s gradient with respect to its tokens; rows past the last end get zeros."""
    _check_kind(experts, 3, "grouped_linear_fp4_grad_input takes a stack of experts and a rank-two gradient.")
    if grad.ndim != 2:
        raise ValueError("grouped_linear_fp4_grad_input takes a stack of experts and a rank-two gradient.")
    _check_ends(group_ends, experts.qdata.shape[0], experts.qdata.device)
    return _grad_input(grad, experts, group_ends)
