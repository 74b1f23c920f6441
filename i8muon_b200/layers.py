"""The layers around the matrices that Muon steps: what makes their gradients.

``linear`` (bias, activation and residual in the product's epilogue), ``layer_norm``, and activations kept in eight bits for the backward pass (``quantise_activation``, ``restore_activation``,
and the ``checkpoint=`` argument of the layers).  The functions take and return torch tensors, work on
the current stream of the tensors' device without synchronising, and are differentiable once, in reverse mode; tensors that
carry a tangent of forward mode are refused.  They run the sm_100a library's kernels; there is no fallback.  The reference
starts at the gradient and has no counterpart.

Eight-bit format: groups of 32 consecutive elements of a row share a power of two, the smallest 2^e with
max|x| <= M 2^e (M = 127 for ``"int8"``, 448 for ``"fp8"``, E4M3; e >= -127), and each element is rounded to the nearest
code, ties to even.  The values that codes stand for are exact in the activation's own type.  A group that holds an
infinity or a NaN reads back as NaN.  An element costs 33/32 bytes.
"""
from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple, Optional

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import native
from .engine import on_device, raw_stream, status_word

__all__ = ["linear", "layer_norm", "quantise_activation", "restore_activation", "QuantisedActivation"]

GROUP = 32
_FORMATS = {None: native.EIGHT_NONE, "int8": native.EIGHT_INT8, "fp8": native.EIGHT_E4M3}
_CODE_TYPES = {native.EIGHT_INT8: torch.int8, native.EIGHT_E4M3: torch.float8_e4m3fn}
_ACTIVATIONS = {None: 0, "relu": 1, "relu2": 2, "gelu": 3, "gelu_tanh": 4, "silu": 5}
_MOST_WIDTH, _MOST_ROWS = native.MAX_LAYER_WIDTH, native.MAX_LAYER_ROWS
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


class QuantisedActivation(NamedTuple):
    """An activation in eight bits: codes (..., 32 ceil(width / 32)) and exponent bytes (..., ceil(width / 32)) of a
    tensor of ``shape`` and ``dtype``."""
    codes: Tensor
    exponents: Tensor
    shape: torch.Size
    dtype: torch.dtype
    checkpoint: str


# ------------------------------------------------------------------ checks
def _format(name, function):
    try:
        return _FORMATS[name]
    except (KeyError, TypeError):
        raise ValueError(f"{function}: checkpoint must be None, 'int8' or 'fp8'") from None


@lru_cache(maxsize=None)
def _is_sm100(index: int) -> bool:
    return torch.cuda.get_device_capability(index)[0] == 10


def _check_device(function, x, *others):
    for t in others:
        if t is not None and t.device != x.device:
            raise ValueError(f"{function}: all tensors must be on one device")
    if not x.is_cuda:
        raise ValueError(f"{function} needs CUDA tensors")
    if not _is_sm100(x.device.index):
        raise ValueError("The i8muon_b200 kernels are built for sm_100a (B200) only.")


def _check_rows(function, x, dtypes=_FLOATS):
    """``x`` as rows of its last dimension: (number of rows, width)."""
    if not isinstance(x, Tensor) or x.ndim < 1:
        raise ValueError(f"{function}: expected a tensor with at least one dimension")
    if x.dtype not in dtypes:
        raise ValueError(f"{function}: the input must be " + " or ".join(str(t).replace("torch.", "") for t in dtypes))
    width = x.shape[-1]
    if width < 1:
        raise ValueError(f"{function}: the last dimension must not be empty")
    rows = x.numel() // width
    if width > _MOST_WIDTH or rows > _MOST_ROWS:
        raise _too_large(function, rows, width)
    return rows, width


def _too_large(function, rows, width):
    return ValueError(f"{function}: {rows} rows of {width} elements are above the limits, {_MOST_ROWS} rows and {_MOST_WIDTH} elements")


def _check_vector(function, name, v, width, dtype):
    if v is not None and (not isinstance(v, Tensor) or v.shape != (width,) or v.dtype != dtype):
        raise ValueError(f"{function}: {name} must be a vector of {width} elements of the input's type")


def _ptr(t: Optional[Tensor]):
    return None if t is None else t.data_ptr()


def _workspace(size, like):
    return like.new_empty((size,), dtype=torch.uint8) if size else None


_STATUS_ADDRESSES: dict = {}      # device index -> address of its status word, which stays


def _status(device) -> int:
    address = _STATUS_ADDRESSES.get(device.index)
    if address is None:
        # the word's first zeros would become part of the graph, and it would hold anything until the first replay
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("linear: make one call on this device before capturing one into a graph")
        address = _STATUS_ADDRESSES.setdefault(device.index, status_word(device).data_ptr())
    return address


def _any_gradient(*tensors) -> bool:
    for t in tensors:
        if t is not None and t.requires_grad:
            return torch.is_grad_enabled()
    return False


def _refuse_tangents(function, *tensors):
    """A dual tensor of forward mode need not require a gradient, and the kernels would drop its tangent: a derivative of zero."""
    if getattr(forward_ad, "_current_level", 0) < 0:      # no level is entered, which is nearly always
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{function} has no forward-mode derivative")


# ------------------------------------------------------- activations in eight bits
def _quantise(x, rows, width, fmt, codes_at, exponents_at):
    """A contiguous ``x`` to codes and exponents at two addresses; its device must be current."""
    native.call("i8m_activation_quant", x.data_ptr(), native.torch_dtype_code(x.dtype), rows, width, fmt, codes_at, exponents_at,
                raw_stream(x.device.index))


def _eight_buffer(like, rows, width):
    """One buffer for what a layer keeps in eight bits, codes first, and the offset of the exponents."""
    groups = -(-width // GROUP)
    return like.new_empty((rows * groups * (GROUP + 1),), dtype=torch.uint8), rows * groups * GROUP


def quantise_activation(x: Tensor, checkpoint: str = "int8") -> QuantisedActivation:
    """``x`` (float32, float16 or bfloat16, any number of rows of its last dimension) in eight bits.  Not
    differentiable: the result carries no graph."""
    fmt = _format(checkpoint, "quantise_activation")
    if fmt == native.EIGHT_NONE:
        raise ValueError("quantise_activation: checkpoint must be 'int8' or 'fp8'")
    rows, width = _check_rows("quantise_activation", x)
    _refuse_tangents("quantise_activation", x)
    _check_device("quantise_activation", x)
    groups = -(-width // GROUP)
    shape = x.shape
    if x.requires_grad:
        x = x.detach()
    x = x.contiguous()
    with on_device(x.device.index):
        codes = x.new_empty((*shape[:-1], groups * GROUP), dtype=_CODE_TYPES[fmt])
        exponents = x.new_empty((*shape[:-1], groups), dtype=torch.uint8)
        if rows:
            _quantise(x, rows, width, fmt, codes.data_ptr(), exponents.data_ptr())
    return QuantisedActivation(codes, exponents, shape, x.dtype, checkpoint)


def restore_activation(q: QuantisedActivation) -> Tensor:
    """The values that ``q`` stands for, as a fresh tensor of the activation's shape and type."""
    if not isinstance(q, QuantisedActivation):
        raise ValueError("restore_activation: expected what quantise_activation returned")
    fmt = _format(q.checkpoint, "restore_activation")
    shape = torch.Size(q.shape)
    if fmt == native.EIGHT_NONE or len(shape) < 1 or shape[-1] < 1 or q.dtype not in _FLOATS:
        raise ValueError("restore_activation: not a quantised activation")
    width = shape[-1]
    groups = -(-width // GROUP)
    if (q.codes.shape != (*shape[:-1], groups * GROUP) or q.codes.dtype != _CODE_TYPES[fmt]
            or q.exponents.shape != (*shape[:-1], groups) or q.exponents.dtype != torch.uint8):
        raise ValueError("restore_activation: codes and exponents do not belong to a tensor of this shape")
    rows = q.exponents.numel() // groups
    if width > _MOST_WIDTH or rows > _MOST_ROWS:
        raise _too_large("restore_activation", rows, width)
    _check_device("restore_activation", q.codes, q.exponents)
    device = q.codes.device
    codes, exponents = q.codes.contiguous(), q.exponents.contiguous()
    if codes.data_ptr() % 16:
        codes = codes.clone()
    with on_device(device.index):
        out = codes.new_empty(shape, dtype=q.dtype)
        if rows:
            native.call("i8m_activation_restore", codes.data_ptr(), exponents.data_ptr(), rows, width, fmt,
                        out.data_ptr(), native.torch_dtype_code(q.dtype), raw_stream(device.index))
    return out


# ------------------------------------------------------------------ layer norm
def _norm_forward(x, weight, bias, eps, fmt, keep):
    """(y, statistics, what is kept in eight bits and the offset of its exponents) of a contiguous ``x``.  Statistics: the
    rows' means and reciprocal deviations, or the latter alone beside eight bits; nothing is kept unless ``keep``."""
    width = x.shape[-1]
    rows, index = x.numel() // width, x.device.index
    with on_device(index):
        y = torch.empty_like(x)
        stats = eight = mean_at = rstd_at = codes_at = exponents_at = None
        offset = 0
        if keep:
            if fmt == native.EIGHT_NONE:
                stats = x.new_empty((2, rows), dtype=torch.float32)
                mean_at = stats.data_ptr()
                rstd_at = mean_at + 4 * rows
            else:
                stats = x.new_empty((rows,), dtype=torch.float32)
                rstd_at = stats.data_ptr()
                eight, offset = _eight_buffer(x, rows, width)
                codes_at = eight.data_ptr()
                exponents_at = codes_at + offset
        if rows:
            native.call("i8m_layer_norm", x.data_ptr(), _ptr(weight), _ptr(bias), y.data_ptr(), mean_at, rstd_at, codes_at,
                        exponents_at, fmt if keep else native.EIGHT_NONE, rows, width, native.torch_dtype_code(x.dtype), eps,
                        raw_stream(index))
    return y, stats, eight, offset


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, fmt):
        x = x.contiguous()
        weight = None if weight is None else weight.contiguous()
        y, stats, eight, offset = _norm_forward(x, weight, None if bias is None else bias.contiguous(), eps, fmt, True)
        ctx.settings = fmt, x.shape, offset
        kept = x if eight is None else eight
        if weight is None:
            ctx.save_for_backward(kept, stats)
        else:
            ctx.save_for_backward(kept, stats, weight)
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():         # a graph of the gradients is asked for: its use is refused, not their value
            return _norm_backward_once(ctx, dy)
        return _norm_backward(ctx, dy)


def _norm_backward(ctx, dy):
    need_x, need_w, need_b = ctx.needs_input_grad[:3]
    fmt, shape, offset = ctx.settings
    kept, stats, *weight = ctx.saved_tensors
    _refuse_tangents("layer_norm", dy)
    width = shape[-1]
    dy = dy.contiguous()
    rows, index = dy.numel() // width, dy.device.index
    with on_device(index):
        make = dy.new_zeros if rows == 0 else dy.new_empty
        dx = make(shape) if need_x else None
        dw = make((width,)) if need_w else None
        db = make((width,)) if need_b else None
        if rows:
            kept_at, stats_at = kept.data_ptr(), stats.data_ptr()
            if fmt == native.EIGHT_NONE:
                at = kept_at, stats_at, stats_at + 4 * rows, None, None
            else:
                at = None, None, stats_at, kept_at, kept_at + offset
            size = native.layer_norm_scratch_bytes(rows, width) if need_w or need_b else 0
            scratch = _workspace(size, dy)
            native.call("i8m_layer_norm_backward", dy.data_ptr(), *at, fmt, weight[0].data_ptr() if weight else None, _ptr(dx),
                        _ptr(dw), _ptr(db), rows, width, native.torch_dtype_code(dy.dtype), _ptr(scratch), size,
                        raw_stream(index))
    return dx, dw, db, None, None


_norm_backward_once = once_differentiable(_norm_backward)


def layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5, *,
               checkpoint: Optional[str] = None) -> Tensor:
    """Layer norm over the last dimension: ``(x - mean) / sqrt(var + eps) * weight + bias``.

    ``x`` in float32, float16 or bfloat16; ``weight`` and ``bias`` (either may be None) are vectors of the same type.
    Statistics and sums are FP32, the result is rounded once.  For the backward pass ``x`` and two statistics per row are
    kept, or, with ``checkpoint="int8"`` or ``"fp8"``, the normalised rows in eight bits and one statistic; the gradients
    are then those of the formula at the kept rows."""
    fmt = _format(checkpoint, "layer_norm")
    _, width = _check_rows("layer_norm", x)
    _check_vector("layer_norm", "weight", weight, width, x.dtype)
    _check_vector("layer_norm", "bias", bias, width, x.dtype)
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError("layer_norm: eps must be >= 0")
    _refuse_tangents("layer_norm", x, weight, bias)
    _check_device("layer_norm", x, weight, bias)
    if _any_gradient(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps, fmt)
    return _norm_forward(x.contiguous(), None if weight is None else weight.contiguous(),
                         None if bias is None else bias.contiguous(), eps, native.EIGHT_NONE, False)[0]


# ---------------------------------------------------------------------- linear
def _linear_forward(x, weight, bias, residual, activation, fmt, keep):
    """(y, the kept pre-activation and, in eight bits, the offset of its exponents) of contiguous tensors; nothing is kept unless
    ``keep``."""
    inner, outer = x.shape[-1], weight.shape[0]
    rows, device = x.numel() // inner, x.device
    with on_device(device.index):
        y = x.new_empty((*x.shape[:-1], outer))
        z = z_at = codes_at = exponents_at = None
        offset = 0
        if keep:
            if fmt == native.EIGHT_NONE:
                z = x.new_empty((rows, -(-outer // 8) * 8))
                z_at = z.data_ptr()
            else:
                z, offset = _eight_buffer(x, rows, outer)
                codes_at = z.data_ptr()
                exponents_at = codes_at + offset
        if rows:
            x_at, w_at = x.data_ptr(), weight.data_ptr()
            size = 0
            if inner % 8 or (x_at | w_at) % 16:
                size = native.linear_workspace_bytes(x_at, w_at, rows, inner, outer)
            workspace = _workspace(size, x)
            native.call("i8m_linear", x_at, w_at, _ptr(bias), _ptr(residual), y.data_ptr(), z_at, codes_at, exponents_at, fmt,
                        activation, rows, inner, outer, native.torch_dtype_code(x.dtype), _ptr(workspace), size, _status(device),
                        raw_stream(device.index))
    return y, z, offset


@lru_cache(maxsize=4096)
def _backward_bytes(dy, x, weight, rows, inner, outer, activation, fmt, dx, dw, db):
    """Workspace of a backward call; dy, x and weight are addresses modulo 16."""
    return native.linear_backward_workspace_bytes(dy, x, weight, rows, inner, outer, activation, fmt, dx, dw, db)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, fmt):
        x, weight = x.contiguous(), weight.contiguous()
        bias = None if bias is None else bias.contiguous()
        residual = None if residual is None else residual.contiguous()
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        keep_z = activation != 0 and (need_x or need_w or need_b)
        y, z, z_offset = _linear_forward(x, weight, bias, residual, activation, fmt, keep_z)
        kept = [weight] if need_x else []
        x_offset = 0
        if need_w:
            if fmt == native.EIGHT_NONE:
                kept.append(x)
            else:
                inner = x.shape[-1]
                rows = x.numel() // inner
                with on_device(x.device.index):
                    eight, x_offset = _eight_buffer(x, rows, inner)
                    if rows:
                        _quantise(x, rows, inner, fmt, eight.data_ptr(), eight.data_ptr() + x_offset)
                kept.append(eight)
        if keep_z:
            kept.append(z)
        ctx.settings = activation, fmt, x.shape, weight.shape, keep_z, x_offset, z_offset
        ctx.save_for_backward(*kept)
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():         # a graph of the gradients is asked for: its use is refused, not their value
            return _linear_backward_once(ctx, dy)
        return _linear_backward(ctx, dy)


def _linear_backward(ctx, dy):
    need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
    activation, fmt, x_shape, w_shape, kept_z, x_offset, z_offset = ctx.settings
    dresidual = dy if need_r else None
    if not (need_x or need_w or need_b):
        return None, None, None, dresidual, None, None
    _refuse_tangents("linear", dy)
    kept = iter(ctx.saved_tensors)
    weight = next(kept) if need_x else None
    x = next(kept) if need_w else None
    z = next(kept) if kept_z else None
    outer, inner = w_shape
    dy = dy.contiguous()
    rows, device = dy.numel() // outer, dy.device
    with on_device(device.index):
        make = dy.new_zeros if rows == 0 else dy.new_empty
        dx = make(x_shape) if need_x else None
        dw = make(w_shape) if need_w else None
        db = make((outer,)) if need_b else None
        if rows:
            dy_at, x_at, w_at, z_at = dy.data_ptr(), _ptr(x), _ptr(weight), _ptr(z)
            # x and z, or their codes and exponents
            x_codes = x_exponents = z_codes = z_exponents = None
            if fmt != native.EIGHT_NONE:
                if need_w:
                    x_at, x_codes, x_exponents = None, x_at, x_at + x_offset
                if kept_z:
                    z_at, z_codes, z_exponents = None, z_at, z_at + z_offset
            size = _backward_bytes(dy_at & 15, (x_at or 0) & 15, (w_at or 0) & 15, rows, inner, outer, activation, fmt, need_x, need_w,
                                   need_b)
            workspace = _workspace(size, dy)
            native.call("i8m_linear_backward", dy_at, x_at, x_codes, x_exponents, w_at, z_at, z_codes, z_exponents, fmt, activation,
                        _ptr(dx), _ptr(dw), _ptr(db), rows, inner, outer, native.torch_dtype_code(dy.dtype), _ptr(workspace), size,
                        _status(device), raw_stream(device.index))
    return dx, dw, db, dresidual, None, None


_linear_backward_once = once_differentiable(_linear_backward)


def linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, *, activation: Optional[str] = None,
           residual: Optional[Tensor] = None, checkpoint: Optional[str] = None) -> Tensor:
    """``act(x @ weight.T + bias) + residual`` in one product.

    ``x`` (..., inner) in float16 or bfloat16, ``weight`` (outer, inner) as ``torch.nn.Linear`` holds it, ``bias`` (outer),
    ``residual`` (..., outer), all of one type.  ``activation``: None, "relu", "relu2" (max(z, 0)^2), "gelu" (with the
    error function), "gelu_tanh" or "silu".  Sums, bias, activation and residual are FP32; the result is rounded once.  Logistic
    functions below 2^-126 are zero: silu below -87.3, where it is -1e-36, and gelu_tanh below -10.

    For the backward pass ``x`` and, with an activation, the pre-activation rounded to the type of ``x`` are kept, or both in
    eight bits with ``checkpoint="int8"`` or ``"fp8"``.  The gradients are those of the formula at what was kept; the
    gradient of the pre-activation is rounded to the type of ``x`` once, as the operand of the two backward products.  A
    pre-activation beyond the type of ``x`` is kept as an infinity (in eight bits within FP32's range); slopes there are 0 and 1,
    and infinite on the right of relu2.

    A device-side wait that runs out is reported through the status word that ``check_status()`` and ``Muon.step()`` read; a
    first call on a device cannot be captured into a graph.  A backward pass is captured together with its forward pass, on
    one stream, when no graph of the same leaves is alive that was built on another stream (autograd would join that stream)."""
    fmt = _format(checkpoint, "linear")
    if activation is not None and not isinstance(activation, str) or activation not in _ACTIVATIONS:
        raise ValueError("linear: activation must be None, 'relu', 'relu2', 'gelu', 'gelu_tanh' or 'silu'")
    rows, inner = _check_rows("linear", x, (torch.float16, torch.bfloat16))
    if not isinstance(weight, Tensor) or weight.ndim != 2 or weight.shape[1] != inner or weight.dtype != x.dtype or weight.shape[0] < 1:
        raise ValueError(f"linear: weight must be a matrix of {inner} columns of the input's type")
    outer = weight.shape[0]
    if outer > _MOST_WIDTH:
        raise _too_large("linear", outer, inner)
    _check_vector("linear", "bias", bias, outer, x.dtype)
    if residual is not None and (not isinstance(residual, Tensor) or residual.shape != (*x.shape[:-1], outer)
                                 or residual.dtype != x.dtype):
        raise ValueError("linear: residual must have the shape and type of the result")
    _refuse_tangents("linear", x, weight, bias, residual)
    _check_device("linear", x, weight, bias, residual)
    if _any_gradient(x, weight, bias, residual):
        return _Linear.apply(x, weight, bias, residual, _ACTIVATIONS[activation], fmt)
    return _linear_forward(x.contiguous(), weight.contiguous(), None if bias is None else bias.contiguous(),
                           None if residual is None else residual.contiguous(), _ACTIVATIONS[activation], native.EIGHT_NONE, False)[0]
