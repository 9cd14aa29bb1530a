"""What the operators around the layer (``norm``, ``tokens``) share: checks of row tensors, their way to the C ABI, and the rule
on stream capture."""
from __future__ import annotations

import contextlib
import functools
from typing import Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from .kernel import _require_cuda

DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}
MAX_TOKENS = 1 << 24


def check_rows(t, name: str) -> Tuple[int, int]:
    """(rows, columns) of a 2-d tensor of bf16, f16 or f32."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype not in DTYPES:
        raise TypeError(f"{name} must be bfloat16, float16 or float32, got {t.dtype}")
    shape = t.shape
    if len(shape) != 2:
        raise ValueError(f"{name} must have two dimensions, got {tuple(shape)}")
    return shape[0], shape[1]


def check_tensor(t, name: str, dtype: torch.dtype, shape: Tuple[int, ...]) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")


def refuse_tangents(*tensors) -> None:
    """Forward-mode derivatives are not available: a tensor that carries a tangent (it need not require a gradient) would come out
    without one, which counts as zero.  Outside of ``forward_ad.dual_level()`` there are none."""
    if forward_ad._current_level < 0:
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("the operators around the layer have no forward-mode derivative: an input carries a tangent")


def check_device(first: torch.Tensor, *tensors) -> torch.device:
    """The CUDA device of ``first``, on which all others must be too.  Every operator passes all its tensors through here, so tangents
    are refused here as well."""
    device = first.device
    for t in tensors:
        if t is not None and t.device != device:
            _require_cuda(input=first, argument=t)
            raise RuntimeError(f"all tensors must live on one device: got {t.device} beside {device}")
    if not first.is_cuda:
        _require_cuda(input=first)
    refuse_tangents(first, *tensors)
    return device


def row_pointer(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """A tensor whose rows the library can read in place and their distance in bytes (0 = dense): ``t`` itself where its rows are
    dense, 16-byte aligned and apart, else a copy.  The caller keeps the tensor until the launch."""
    size = t.element_size()
    if t.is_contiguous():
        return (t if t.data_ptr() % 16 == 0 else t.clone()), 0
    pitch = t.stride(0) * size
    if t.stride(1) == 1 and t.stride(0) >= t.shape[1] and pitch % 16 == 0 and t.data_ptr() % 16 == 0:
        return t, pitch
    return t.contiguous(), 0


def dense(t: torch.Tensor, align: int = 4) -> torch.Tensor:
    """``t`` if it is contiguous and its address a multiple of ``align``, else a copy."""
    if not t.is_contiguous():
        return t.contiguous()
    return t if t.data_ptr() % align == 0 else t.clone()


_HERE = contextlib.nullcontext()


def on_device(device: torch.device):
    """Context in which ``device`` is the current one."""
    return _HERE if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def stream_of(device: torch.device) -> int:
    """The device's current stream as the C ABI takes it.  (torch.cuda.current_stream builds a Stream object for it: 2.3 us, of
    the ~10 that a small call takes on the host; this call 0.1.)"""
    return torch._C._cuda_getCurrentRawStream(device.index)


class _FirstDerivative(torch.autograd.Function):
    """Passes gradients on; differentiating them raises."""

    @staticmethod
    def forward(ctx, anchor, *grads):
        return tuple(None if g is None else g.view_as(g) for g in grads)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("the operators around the layer are differentiable once: a second derivative is not available")


def differentiable_once(backward):
    """For the backward pass of an autograd function: where gradients are recorded (``create_graph=True``) its results raise when
    they are differentiated in turn.  (torch's own ``once_differentiable`` does so only where the incoming gradients
    require one; the results of a constant gradient would count as constants of the inputs.)"""
    @functools.wraps(backward)
    def call(ctx, *grads):
        refuse_tangents(*grads)
        if not torch.is_grad_enabled():
            return backward(ctx, *grads)
        with torch.no_grad():
            results = backward(ctx, *grads)
        results = results if isinstance(results, tuple) else (results,)
        if all(r is None for r in results):
            return results
        return _FirstDerivative.apply(torch.empty(0, requires_grad=True), *results)
    return call


def records_graph(instead: str, *tensors) -> bool:
    """Whether a call on these tensors has to record an autograd node.  During stream capture that is refused: where an eager
    graph over the same leaves is alive, their accumulation nodes belong to another stream than the captured one, and running
    them under capture ends the process.  ``instead`` names the function that computes the gradient explicitly."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                refuse_capture(instead, t.device)
                return True
    return False


def refuse_capture(instead: str, device: torch.device) -> None:
    """Raises if the device's current stream is being captured.  In a backward pass that is the stream of the forward call: autograd
    makes it current while it runs the node."""
    with on_device(device):
        capturing = torch.cuda.is_current_stream_capturing()
    if capturing:
        raise RuntimeError("autograd is not available during stream capture: capture the call under torch.no_grad() and "
                           f"its gradient as {instead}(...)")
