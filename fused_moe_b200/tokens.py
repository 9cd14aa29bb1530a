"""Tokens sorted by expert and back, for experts that are the user's own products (training, other weights than the layer's),
and the weights of the selected experts; all with their gradients.

    idx, _  = kernel.route(logits, bias, scale)                 # selects, no gradient
    weights = route_weights(logits, idx, scale)                 # the selection's weights, differentiable in the logits
    plan    = sort_tokens(idx, E_local, offset, align=128)
    xs      = gather_tokens(x, plan)                            # rows of expert e: plan.offsets[e] .. + plan.counts[e]
    out     = combine_tokens(experts(xs, plan), weights, plan)

``kernel`` does all of this inside one call for its own FP8 experts (the reference: solution/python/pure_triton_impl.py:474-551
sorts, :1758-1821 reduces); the reference has no gradient.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _lib
from .kernel import E_GLOBAL, TOP_K, _host_scalar
from .rows import DTYPES, MAX_TOKENS, check_device, check_rows, check_tensor, dense, differentiable_once, on_device, \
    records_graph, refuse_capture, refuse_tangents, row_pointer, stream_of


class TokenSort(NamedTuple):
    """Where each (token, k) pair of a batch goes.  Device tensors of int32; nothing here was read by the host.

    counts [E]          pairs of each local expert (those without a row among them, see ``rows``)
    offsets [E + 1]     first row of each expert's segment, a multiple of ``align``, and the end of the last; at most ``rows``
    row_pairs [rows]    pair t * K + k of each row, -1 for a row without one
    scatter_map [T, K]  row of each pair, -1 for a pair without one
    rows                capacity: rows of a sorted batch
    """

    counts: torch.Tensor
    offsets: torch.Tensor
    row_pairs: torch.Tensor
    scatter_map: torch.Tensor
    rows: int
    align: int


def _selection(topk_idx) -> tuple:
    if not isinstance(topk_idx, torch.Tensor):
        raise TypeError("topk_idx must be a torch.Tensor")
    if topk_idx.dtype is not torch.int32:
        raise TypeError(f"topk_idx must be torch.int32, got {topk_idx.dtype}")
    shape = topk_idx.shape
    if len(shape) != 2 or not 1 <= shape[1] <= TOP_K or shape[0] > MAX_TOKENS:
        raise ValueError(f"topk_idx must be [T, K] with K in 1..{TOP_K} and T <= {MAX_TOKENS}, got {tuple(shape)}")
    return shape[0], shape[1]


def sort_tokens(topk_idx: torch.Tensor, E_local: int, local_expert_offset=0, align: int = 1,
                rows: Optional[int] = None) -> TokenSort:
    """Sorts the pairs of ``topk_idx`` [T, K] int32 (K <= 8, global expert ids) stably by local expert: row of a pair = start of
    its expert's segment + earlier pairs of that expert.  Segments start at multiples of ``align``.  Ids outside
    [local_expert_offset, local_expert_offset + E_local) take no part; -1 marks the padding of a batch.  A token may name an
    expert twice.

    ``rows`` is the capacity of the sorted batch, on which all shapes depend; None = what any routing fits into (T * K, or
    (T * K / align + E_local) * align).  A pair whose row would be ``rows`` or more gets none (its token does without that
    expert, ``counts`` still counts it), so a smaller capacity needs no host synchronisation.  Scratch is allocated per
    call: calls on different streams, or in different graphs, share nothing."""
    T, K = _selection(topk_idx)
    offset = _host_scalar(local_expert_offset, int)
    if not 1 <= E_local <= E_GLOBAL:
        raise ValueError(f"E_local must be in 1..{E_GLOBAL}, got {E_local}")
    if offset < 0 or offset + E_local > E_GLOBAL:
        raise ValueError(f"local_expert_offset {offset} with {E_local} local experts exceeds {E_GLOBAL} experts")
    if align < 1 or T * K + E_local * (align - 1) > _lib.TOKEN_MAX_ROWS:
        raise ValueError(f"align must be at least 1 and the padded rows at most {_lib.TOKEN_MAX_ROWS}")
    if rows is None:
        rows = T * K if align == 1 else (T * K // align + min(E_local, T * K)) * align
    if not 0 <= rows <= _lib.TOKEN_MAX_ROWS:
        raise ValueError(f"rows must be in 0..{_lib.TOKEN_MAX_ROWS}")
    device = check_device(topk_idx)
    idx = dense(topk_idx)
    lib = _lib.load()
    need = C.c_size_t(0)
    _lib.check(lib.b200moe_token_sort_scratch_bytes(T, K, E_local, C.byref(need)), "b200moe_token_sort_scratch_bytes")
    ints = topk_idx.new_empty
    plan = TokenSort(ints(E_local), ints(E_local + 1), ints(rows), ints(T, K), rows, align)
    scratch = ints(need.value // 4) if need.value else None   # a small batch needs none
    with on_device(device):
        _lib.check(lib.b200moe_token_sort(idx.data_ptr(), T, K, E_local, offset, align, rows,
                                          None if scratch is None else scratch.data_ptr(), need.value,
                                          plan.counts.data_ptr(), plan.offsets.data_ptr(), plan.row_pairs.data_ptr(),
                                          plan.scatter_map.data_ptr(), stream_of(device)),
                   "b200moe_token_sort")
    return plan


def _check_plan(plan) -> None:
    """A plan may have been put together by hand or from several: the arrays that the kernels index are checked on every call.
    (Their entries are not read here; the kernels take one that lies outside the buffers for -1.)"""
    if not isinstance(plan, TokenSort):
        raise TypeError("plan must be a TokenSort")
    scatter_map, row_pairs = plan.scatter_map, plan.row_pairs
    if not isinstance(scatter_map, torch.Tensor) or scatter_map.dtype is not torch.int32:
        raise TypeError("plan.scatter_map must be an int32 tensor")
    if not isinstance(row_pairs, torch.Tensor) or row_pairs.dtype is not torch.int32:
        raise TypeError("plan.row_pairs must be an int32 tensor")
    if not (scatter_map.is_contiguous() and row_pairs.is_contiguous()):
        raise ValueError("plan.scatter_map and plan.row_pairs must be contiguous")
    shape = scatter_map.shape
    if len(shape) != 2 or not 1 <= shape[1] <= TOP_K or shape[0] > MAX_TOKENS:
        raise ValueError(f"plan.scatter_map must be [T, K] with K in 1..{TOP_K} and T <= {MAX_TOKENS}, got {tuple(shape)}")
    if row_pairs.shape != (plan.rows,):
        raise ValueError(f"plan.row_pairs must have plan.rows = {plan.rows} entries, got {tuple(row_pairs.shape)}")


def _check_batch(t, name: str, plan: TokenSort, rows: int) -> int:
    n, columns = check_rows(t, name)
    if n != rows:
        raise ValueError(f"{name} must have {rows} rows, got {n}")
    if columns == 0 or columns * t.element_size() % 16 or columns > 1 << 24:
        raise ValueError(f"a row of {name} must be a multiple of 16 bytes, got {columns} columns of {t.dtype}")
    check_device(t, plan.scatter_map, plan.row_pairs)
    return columns


def _gather(x: torch.Tensor, plan_rows: int, row_pairs: torch.Tensor, scatter_map: torch.Tensor) -> torch.Tensor:
    (T, K), columns, device = scatter_map.shape, x.shape[1], x.device
    out = x.new_empty(plan_rows, columns)
    xr, pitch = row_pointer(x)
    with on_device(device):
        _lib.check(_lib.load().b200moe_token_gather(xr.data_ptr(), pitch, DTYPES[x.dtype], T, K, columns, plan_rows,
                                                    row_pairs.data_ptr(), scatter_map.data_ptr(), out.data_ptr(),
                                                    stream_of(device)), "b200moe_token_gather")
    return out


def _combine(rows: torch.Tensor, weights: Optional[torch.Tensor], scatter_map: torch.Tensor) -> torch.Tensor:
    (T, K), columns, device = scatter_map.shape, rows.shape[1], rows.device
    out = rows.new_empty(T, columns)
    rr, pitch = row_pointer(rows)
    w = None if weights is None else dense(weights)
    with on_device(device):
        _lib.check(_lib.load().b200moe_token_combine(rr.data_ptr(), pitch, DTYPES[rows.dtype],
                                                     None if w is None else w.data_ptr(), T, K, columns, rows.shape[0],
                                                     scatter_map.data_ptr(), out.data_ptr(),
                                                     stream_of(device)),
                   "b200moe_token_combine")
    return out


def _combine_backward(grad, rows, weights, row_pairs, scatter_map, need_rows: bool, need_weights: bool):
    """``rows`` may be None where the weights' gradient is not needed."""
    (T, K), columns, device, n = scatter_map.shape, grad.shape[1], grad.device, row_pairs.shape[0]
    grad_rows = grad.new_empty(n, columns) if need_rows else None
    grad_weights = weights.new_empty(T, K) if need_weights else None
    gr, g_pitch = row_pointer(grad)
    rr, r_pitch = (None, 0) if rows is None else row_pointer(rows)
    w = dense(weights)
    with on_device(device):
        _lib.check(_lib.load().b200moe_token_combine_backward(
            gr.data_ptr(), g_pitch, None if rr is None else rr.data_ptr(), r_pitch, DTYPES[grad.dtype], w.data_ptr(), T, K,
            columns, n, row_pairs.data_ptr(), scatter_map.data_ptr(), None if grad_rows is None else grad_rows.data_ptr(),
            None if grad_weights is None else grad_weights.data_ptr(), stream_of(device)),
            "b200moe_token_combine_backward")
    return grad_rows, grad_weights


class _GatherTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, plan):
        ctx.save_for_backward(plan.scatter_map)
        return _gather(x, plan.rows, plan.row_pairs, plan.scatter_map)

    @staticmethod
    @differentiable_once
    def backward(ctx, grad):
        refuse_capture("gather_tokens_backward", grad.device)
        return _combine(grad, None, *ctx.saved_tensors), None


class _CombineTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, plan):
        # the rows are kept only for the weights' gradient
        ctx.save_for_backward(rows if ctx.needs_input_grad[1] else None, weights, plan.row_pairs, plan.scatter_map)
        return _combine(rows, weights, plan.scatter_map)

    @staticmethod
    @differentiable_once
    def backward(ctx, grad):
        refuse_capture("combine_tokens_backward", grad.device)
        rows, weights, row_pairs, scatter_map = ctx.saved_tensors
        return (*_combine_backward(grad, rows, weights, row_pairs, scatter_map, *ctx.needs_input_grad[:2]), None)


def gather_tokens(x: torch.Tensor, plan: TokenSort) -> torch.Tensor:
    """[plan.rows, n]: row r is x[t] for the pair (t, k) of row r, and zero for a row without a pair.  x [T, n] bf16, f16 or f32 with
    rows of whole 16 bytes; row-strided input is read in place.  Differentiable once in x: the gradient of a token is the sum
    of its rows' gradients, in float32, in the order of k."""
    _check_plan(plan)
    _check_batch(x, "x", plan, plan.scatter_map.shape[0])
    if records_graph("gather_tokens_backward", x):
        return _GatherTokens.apply(x, plan)
    return _gather(x, plan.rows, plan.row_pairs, plan.scatter_map)


def gather_tokens_backward(grad: torch.Tensor, plan: TokenSort) -> torch.Tensor:
    """Gradient [T, n] of the x of ``gather_tokens`` from that of its result; can be captured into a CUDA graph."""
    _check_plan(plan)
    _check_batch(grad, "grad", plan, plan.rows)
    return _combine(grad, None, plan.scatter_map)


def _check_weights(weights, plan: TokenSort, first: torch.Tensor) -> None:
    check_tensor(weights, "topk_weights", torch.float32, plan.scatter_map.shape)
    check_device(first, weights)


def combine_tokens(rows: torch.Tensor, topk_weights: torch.Tensor, plan: TokenSort) -> torch.Tensor:
    """[T, n]: out[t] = sum over k of topk_weights[t, k] * rows[row of (t, k)], float32 sums in the order of k, rounded once to the
    type of ``rows``; zero for a token without a row.  rows [plan.rows, n] bf16, f16 or f32, topk_weights [T, K] f32.
    Rows without a pair are not read.  Differentiable once in both: rows without a pair get gradient 0, so do the weights of
    pairs without a row."""
    _check_plan(plan)
    _check_batch(rows, "rows", plan, plan.rows)
    _check_weights(topk_weights, plan, rows)
    if records_graph("combine_tokens_backward", rows, topk_weights):
        return _CombineTokens.apply(rows, topk_weights, plan)
    return _combine(rows, topk_weights, plan.scatter_map)


def combine_tokens_backward(grad: torch.Tensor, rows: torch.Tensor, topk_weights: torch.Tensor, plan: TokenSort):
    """Gradients (grad_rows, grad_weights) of ``combine_tokens`` from that of its result, in one pass over the rows; can be
    captured into a CUDA graph.  The same call gives the same bits; grad_weights may differ in its last ones between a batch of at
    most as many tokens as the GPU has SMs and a larger one (more threads share a row's sum)."""
    _check_plan(plan)
    _check_batch(grad, "grad", plan, plan.scatter_map.shape[0])
    check_tensor(rows, "rows", grad.dtype, (plan.rows, grad.shape[1]))
    check_device(grad, rows)
    _check_weights(topk_weights, plan, grad)
    return _combine_backward(grad, rows, topk_weights, plan.row_pairs, plan.scatter_map, True, True)


def _check_logits(routing_logits, topk_idx) -> tuple:
    T, K = _selection(topk_idx)
    check_tensor(routing_logits, "routing_logits", torch.float32, (T, E_GLOBAL))
    check_device(routing_logits, topk_idx)
    return T, K


def _route_weights(logits, idx, scale: float) -> torch.Tensor:
    T, K = idx.shape
    out = logits.new_empty(T, K)
    logits, idx = dense(logits), dense(idx)
    with on_device(logits.device):
        _lib.check(_lib.load().b200moe_route_weights(logits.data_ptr(), idx.data_ptr(), T, K, scale, out.data_ptr(),
                                                     stream_of(logits.device)),
                   "b200moe_route_weights")
    return out


def _route_weights_backward(logits, idx, grad, scale: float) -> torch.Tensor:
    T, K = idx.shape
    out = logits.new_empty(T, E_GLOBAL)
    logits, idx, grad = dense(logits), dense(idx), dense(grad)
    with on_device(logits.device):
        _lib.check(_lib.load().b200moe_route_weights_backward(logits.data_ptr(), idx.data_ptr(), grad.data_ptr(), T, K, scale,
                                                              out.data_ptr(),
                                                              stream_of(logits.device)),
                   "b200moe_route_weights_backward")
    return out


class _RouteWeights(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, idx, scale):
        ctx.save_for_backward(logits, idx)
        ctx.scale = scale
        return _route_weights(logits, idx, scale)

    @staticmethod
    @differentiable_once
    def backward(ctx, grad):
        refuse_capture("route_weights_backward", grad.device)
        return _route_weights_backward(*ctx.saved_tensors, grad, ctx.scale), None, None


def _scale(x) -> float:
    """``routed_scaling_factor`` as a number.  A tensor's own derivative is not computed and must not get lost."""
    if torch.is_tensor(x):
        refuse_tangents(x)
        if x.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("routed_scaling_factor has no gradient here: pass a number or a detached tensor")
    return _host_scalar(x, float)


def route_weights(routing_logits: torch.Tensor, topk_idx: torch.Tensor, routed_scaling_factor) -> torch.Tensor:
    """[T, K] float32: the weights s_k / (sum_j s_j + 1e-20) * routed_scaling_factor, s = sigmoid(logit), of the experts that
    ``topk_idx`` [T, K] int32 (K <= 8) names; for the selection of ``kernel.route`` these are its weights, bit for bit.  Ids
    outside 0..255 (-1 for the padding of a batch) have weight 0 and take no part; a NaN logit makes its token's weights NaN
    (``route`` takes it for a large one).  Differentiable once in the logits [T, 256]
    float32; the selection itself, and the bias that shaped it, have no gradient, and a scaling factor that requires one is
    refused."""
    _check_logits(routing_logits, topk_idx)
    scale = _scale(routed_scaling_factor)
    if records_graph("route_weights_backward", routing_logits):
        return _RouteWeights.apply(routing_logits, topk_idx, scale)
    return _route_weights(routing_logits, topk_idx, scale)


def route_weights_backward(routing_logits: torch.Tensor, topk_idx: torch.Tensor, grad_weights: torch.Tensor,
                           routed_scaling_factor) -> torch.Tensor:
    """Gradient [T, 256] of the logits of ``route_weights`` from that of its result; can be captured into a CUDA graph."""
    T, K = _check_logits(routing_logits, topk_idx)
    check_tensor(grad_weights, "grad_weights", torch.float32, (T, K))
    check_device(routing_logits, grad_weights)
    return _route_weights_backward(routing_logits, topk_idx, grad_weights, _scale(routed_scaling_factor))
