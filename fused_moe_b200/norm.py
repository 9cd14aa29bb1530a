"""Residual addition and RMS norm in front of the layer.

``add_rms_norm_quantize`` goes from the residual stream to the ``hidden_states`` / ``hidden_states_scale`` pair that
``kernel`` takes in one launch; ``add_rms_norm`` is the same norm for training, differentiable in all three inputs.  Both follow
  r = x + residual, rounded to the residual's type        y = r * weight / sqrt(mean(r^2) + eps)
with float32 arithmetic on the rounded r.  The squares of a row have to stay in float32's range: above about 1e17 per element
their sum is infinite and y is 0; under 1e-19 they are 0, which is nothing beside an ordinary eps, but leaves ``eps=0`` without
a norm.  The reference takes quantised activations as given and has no such operator.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .rows import DTYPES, MAX_TOKENS, check_device, check_rows, check_tensor, dense, differentiable_once, on_device, \
    records_graph, refuse_capture, row_pointer, stream_of

QBLOCK = 128
_FP8 = torch.float8_e4m3fn


def _check(x, residual, weight, eps, multiple: int, names=("x", "residual")) -> Tuple[int, int]:
    T, columns = check_rows(x, names[0])
    if not 0 < columns <= _lib.NORM_MAX_COLUMNS or columns % multiple:
        raise ValueError(f"{names[0]} must have a multiple of {multiple} columns, at most {_lib.NORM_MAX_COLUMNS}, got "
                         f"{columns}")
    if T > MAX_TOKENS:
        raise ValueError(f"{names[0]} must have at most {MAX_TOKENS} rows")
    if residual is not None:
        wide = isinstance(residual, torch.Tensor) and residual.dtype is torch.float32
        check_tensor(residual, names[1], torch.float32 if wide else x.dtype, (T, columns))
    if not isinstance(weight, torch.Tensor) or (weight.dtype is not x.dtype and weight.dtype is not torch.float32):
        raise TypeError(f"weight must be a tensor of the type of {names[0]} or float32")
    check_tensor(weight, "weight", weight.dtype, (columns,))
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    return T, columns


def _forward(x, residual, weight, eps, stream, y, q, scale) -> None:
    T, columns = x.shape
    if T == 0:
        return
    xr, x_pitch = row_pointer(x)
    rr, r_pitch = (None, 0) if residual is None else row_pointer(residual)
    w = dense(weight, 16)
    device = x.device
    with on_device(device):
        _lib.check(_lib.load().b200moe_add_rms_norm(
            xr.data_ptr(), x_pitch, DTYPES[x.dtype], None if rr is None else rr.data_ptr(), r_pitch,
            DTYPES[x.dtype if rr is None else rr.dtype], w.data_ptr(), DTYPES[w.dtype], T, columns, eps,
            None if rr is None else stream.data_ptr(), None if y is None else y.data_ptr(),
            None if q is None else q.data_ptr(), None if scale is None else scale.data_ptr(),
            stream_of(device)), "b200moe_add_rms_norm")


def _backward(grad_y, grad_stream, stream, weight, eps, need_x: bool, need_residual: bool, need_weight: bool):
    """Gradients of x, residual and weight, those not needed None.  Where x and the residual have one type their gradients are
    one tensor."""
    T, columns = stream.shape
    device = stream.device
    one = grad_y.dtype is stream.dtype
    grad_x = grad_y.new_empty(T, columns) if need_x or (one and need_residual) else None
    grad_residual = grad_x if one else stream.new_empty(T, columns) if need_residual else None
    grad_weight = None
    if T == 0:
        grad_weight = torch.zeros(columns, dtype=weight.dtype, device=device) if need_weight else None
    else:
        partial = None
        if need_weight:
            grad_weight = weight.new_empty(columns)
            partial = weight.new_empty(min(T, _lib.NORM_PARTIAL_ROWS), columns, dtype=torch.float32)
        gy, gy_pitch = row_pointer(grad_y)
        gs, gs_pitch = (None, 0) if grad_stream is None else row_pointer(grad_stream)
        rr, r_pitch = row_pointer(stream)
        w = dense(weight, 16)
        with on_device(device):
            _lib.check(_lib.load().b200moe_add_rms_norm_backward(
                gy.data_ptr(), gy_pitch, DTYPES[gy.dtype], None if gs is None else gs.data_ptr(), gs_pitch, rr.data_ptr(),
                r_pitch, DTYPES[rr.dtype], w.data_ptr(), DTYPES[w.dtype], T, columns, eps,
                None if grad_x is None else grad_x.data_ptr(),
                None if one or grad_residual is None else grad_residual.data_ptr(),
                None if grad_weight is None else grad_weight.data_ptr(), None if partial is None else partial.data_ptr(),
                stream_of(device)), "b200moe_add_rms_norm_backward")
    return grad_x if need_x else None, grad_residual if need_residual else None, grad_weight


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        y = x.new_empty(*x.shape)
        stream = None if residual is None else residual.new_empty(*x.shape)
        _forward(x, residual, weight, eps, stream, y, None, None)
        ctx.save_for_backward(x if residual is None else stream, weight)
        ctx.eps, ctx.x_dtype = eps, x.dtype
        ctx.set_materialize_grads(False)
        return y if residual is None else (y, stream)

    @staticmethod
    @differentiable_once
    def backward(ctx, grad_y, grad_stream=None):
        stream, weight = ctx.saved_tensors
        refuse_capture("add_rms_norm_backward", stream.device)
        need_x, need_residual, need_weight = ctx.needs_input_grad[:3]
        if grad_y is None:   # only the residual stream was used: it passes its gradient on
            if grad_stream is None:
                return None, None, None, None
            grad_x = grad_stream.to(ctx.x_dtype) if need_x else None
            return grad_x, grad_stream if need_residual else None, None, None
        return (*_backward(grad_y, grad_stream, stream, weight, ctx.eps, need_x, need_residual, need_weight), None)


def add_rms_norm(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor,
                 eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, r): the normalised rows in the type of ``x`` and the residual stream after the addition in the type of ``residual``.
    ``residual=None`` is the first norm of a model: r is then ``x`` itself.

    x [T, n] bf16, f16 or f32, n a multiple of 8 up to 16384 · residual [T, n] and weight [n] each of x's type or
    f32.  Row-strided inputs are read in place.  Differentiable once in x, residual and weight; the backward pass saves r and
    the weight only, and its sums have a fixed order: the same call gives the same bits.  A token's results do not depend on
    its neighbours, but y may differ in its last bit between a batch of at most 1024 tokens and a larger one (rows of 520 to 8192
    columns: the squares are added by another number of threads).  During stream capture a call that would record a gradient is
    refused (``add_rms_norm_backward`` is the explicit form)."""
    T, columns = _check(x, residual, weight, eps, 8)
    check_device(x, residual, weight)
    if records_graph("add_rms_norm_backward", x, residual, weight):
        if residual is None:
            return _AddRmsNorm.apply(x, None, weight, eps), x
        return _AddRmsNorm.apply(x, residual, weight, eps)
    y = x.new_empty(T, columns)
    stream = x if residual is None else residual.new_empty(T, columns)
    _forward(x, residual, weight, eps, stream, y, None, None)
    return y, stream


def add_rms_norm_backward(grad_y: torch.Tensor, grad_stream: Optional[torch.Tensor], stream: torch.Tensor,
                          weight: torch.Tensor, eps: float = 1e-6):
    """Gradients (grad_x, grad_residual, grad_weight) of ``add_rms_norm`` from those of its results: ``grad_y`` and, unless
    None, ``grad_stream``; ``stream`` is the r that the forward call returned.  grad_x has the type of ``grad_y``,
    grad_residual that of ``stream`` (the same tensor where the types are equal), grad_weight that of ``weight``.  It
    runs no autograd and allocates nothing but its results and scratch, so it can be captured into a CUDA graph."""
    if not isinstance(stream, torch.Tensor):
        raise TypeError("stream must be a torch.Tensor")
    shape = _check(grad_y, stream, weight, eps, 8, ("grad_y", "stream"))
    if grad_stream is not None:
        check_tensor(grad_stream, "grad_stream", stream.dtype, shape)
    check_device(grad_y, stream, weight, grad_stream)
    return _backward(grad_y, grad_stream, stream, weight, eps, True, True, True)


def add_rms_norm_quantize(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-6, *,
                          residual_out: Optional[torch.Tensor] = None, with_normed: bool = False):
    """(q, scales, r) or, ``with_normed``, (q, scales, r, y): residual addition, RMS norm and the layer's quantisation in one launch.

    q [T, n] e4m3 and scales [n / 128, T] float32 are the ``hidden_states`` / ``hidden_states_scale`` of ``kernel`` (n = 7168), by
    the rule of ``quantize_activations`` on the float32 y; r is the residual stream after the addition; y the normalised rows in
    the type of ``x``, which the router's product reads.  Between batches of at most 1024 tokens and larger ones a scale may differ
    in its last bit, and so a value at the border of two e4m3 steps by one of them.  Arguments as for ``add_rms_norm`` with n a multiple of 128.
    ``residual_out`` [T, n] of the residual's type receives r and may be ``residual`` itself.  Not differentiable: with gradients
    enabled, an input that requires one is refused."""
    T, columns = _check(x, residual, weight, eps, QBLOCK)
    check_device(x, residual, weight)
    if (T and (x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad))
            and torch.is_grad_enabled()):
        # r is the residual stream that the rest of the model builds on: without a graph, everything below it would stay without
        # a gradient.  (An empty batch has none to lose.)
        raise RuntimeError("add_rms_norm_quantize is not differentiable: call it under torch.no_grad(), or add_rms_norm for "
                           "gradients")
    if residual is None:
        if residual_out is not None:
            raise ValueError("residual_out needs a residual")
        stream = x
    elif residual_out is None:
        stream = residual.new_empty(T, columns)
    else:
        stream = residual_out
        check_tensor(stream, "residual_out", residual.dtype, (T, columns))
        check_device(x, stream)
        if not stream.is_contiguous() or stream.data_ptr() % 16:
            raise ValueError("residual_out must be contiguous and 16-byte aligned")
        if stream.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("residual_out is overwritten and must not require a gradient")
        for name, t in (("x", x), ("residual", residual), ("weight", weight)):
            same = t.data_ptr() == stream.data_ptr() and t.dtype is stream.dtype and t.is_contiguous() and t is not weight
            if not same and _overlap(t, stream):
                raise ValueError(f"residual_out overlaps {name} without being it")
    q = x.new_empty(T, columns, dtype=_FP8)
    scale = x.new_empty(columns // QBLOCK, T, dtype=torch.float32)
    y = x.new_empty(T, columns) if with_normed else None
    _forward(x, residual, weight, eps, stream, y, q, scale)
    if residual_out is not None:
        torch.autograd.graph.increment_version(residual_out)   # who saved its old values for a gradient learns of the write
    return (q, scale, stream, y) if with_normed else (q, scale, stream)


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the address ranges of two tensors share a byte."""
    def span(t):
        if t.numel() == 0:
            return t.data_ptr(), t.data_ptr()
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1
