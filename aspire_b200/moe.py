"""Tokens to experts and back: router top-k, sort by expert, dispatch, combine.

A sparse feed-forward layer around the experts' products of
:mod:`aspire_b200.quant`::

    weights, experts, order = moe_route(router_logits, top_k)
    rows = moe_dispatch(x, order)                       # sorted by expert
    h = w4_expert_swiglu(rows, order.offsets, *gate_up)
    y = w4_expert_linear(h, order.offsets, *down)
    x = moe_combine(y, weights, order, residual=x)

A slot is a (token, choice) pair, numbered ``token * top_k + choice``.  Nothing
here reads a size back from the device, so a step can be captured in a CUDA
graph.  ``moe_route`` (its weights), ``moe_dispatch`` and ``moe_combine`` have
gradients; every sum runs in fp32 in a fixed order, so results repeat bit by
bit.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _capi

_TYPES = {torch.float32: _capi.T_F32, torch.bfloat16: _capi.T_BF16, torch.float16: _capi.T_F16}


class ExpertOrder(NamedTuple):
    """The stable sort of the slots by expert.

    ``position`` int32 ``[tokens, top_k]``: a slot's sorted row, -1 without an
    expert.  ``source`` int32 ``[tokens * top_k]``: the slot of a sorted row,
    -1 past the last one.  ``offsets`` int32 ``[experts + 1]``: expert e's rows
    are ``offsets[e] .. offsets[e + 1]``."""

    position: torch.Tensor
    source: torch.Tensor
    offsets: torch.Tensor


def _run_route(logits, experts, num_experts, top_k, renormalize):
    given = logits if logits is not None else experts
    tokens, dev = given.shape[0], given.device
    weights = None
    i32 = dict(dtype=torch.int32, device=dev)
    if logits is not None:
        weights = torch.empty(tokens, top_k, dtype=torch.float32, device=dev)
        experts = torch.empty(tokens, top_k, **i32)
    position = torch.empty(tokens, top_k, **i32)
    source = torch.empty(tokens * top_k, **i32)
    offsets = torch.empty(num_experts + 1, **i32)
    ws, need = None, 0
    if tokens * top_k > 4096:  # fewer never need one
        need = _capi.load_library().aspire_moe_route_workspace(tokens, num_experts, top_k)
        ws = torch.empty(need // 4, **i32) if need else None
    _capi.call("aspire_moe_route", _capi.AspireMoeRouteArgs(
        None if logits is None else logits.data_ptr(), 0 if logits is None else _TYPES[logits.dtype],
        0 if logits is None else logits.stride(0), tokens, num_experts, top_k, renormalize,
        None if weights is None else weights.data_ptr(), experts.data_ptr(), position.data_ptr(), source.data_ptr(),
        offsets.data_ptr(), None if ws is None else ws.data_ptr(), need), dev)
    return weights, experts, ExpertOrder(position, source, offsets)


class _RouteWeights(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_k, renormalize, rest):
        # Only the weights have a gradient; the integers go out by `rest`.
        weights, experts, order = _run_route(logits, None, logits.shape[1], top_k, renormalize)
        rest += (experts, order)
        ctx.renormalize = renormalize
        ctx.logits_dtype, ctx.shape = logits.dtype, logits.shape
        if renormalize:
            ctx.save_for_backward(weights, experts)
        else:
            ctx.save_for_backward(weights, experts, logits)
        return weights

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_weights):
        weights, experts, *rest = ctx.saved_tensors
        grad = torch.empty(ctx.shape, dtype=ctx.logits_dtype, device=weights.device)
        if grad.numel():
            g = grad_weights
            if g.dtype != torch.float32 or not g.is_contiguous():
                g = g.to(torch.float32).contiguous()
            _capi.call("aspire_moe_route_grad", _capi.AspireMoeRouteGradArgs(
                rest[0].data_ptr() if rest else None, _TYPES[ctx.logits_dtype], rest[0].stride(0) if rest else 0,
                weights.data_ptr(), experts.data_ptr(), g.data_ptr(), *ctx.shape, weights.shape[1], ctx.renormalize,
                grad.data_ptr()), weights.device)
        return grad, None, None, None


def moe_route(logits: torch.Tensor, top_k: int, *,
              renormalize: bool = True) -> tuple[torch.Tensor, torch.Tensor, ExpertOrder]:
    """The ``top_k`` experts of every token from the router's ``logits``
    ``[tokens, experts]`` (fp32, bf16 or fp16), their weights and the sort of
    the slots by expert (C ABI ``aspire_moe_route``).

    Returns ``(weights fp32 [tokens, top_k], experts int32 [tokens, top_k],
    order)``.  Equal logits go to the lowest expert.  Weights are the softmax
    over the chosen experts or, without ``renormalize``, over all of them.  A
    NaN or -inf logit is never chosen; a row with fewer than ``top_k`` others
    (a padding row: all -inf) has expert -1 and weight 0 for the rest."""
    shape = logits.shape
    if len(shape) != 2 or logits.dtype not in _TYPES or not logits.is_cuda:
        raise ValueError("logits must be a [tokens, experts] CUDA tensor of float32, bfloat16 or float16")
    if not 1 <= shape[1] <= 512:
        raise ValueError("between 1 and 512 experts are supported")
    if not 1 <= top_k <= min(32, shape[1]):
        raise ValueError("top_k must be between 1 and min(32, experts)")
    if logits.stride(1) != 1 and shape[1] > 1 and shape[0]:
        raise ValueError("logits need contiguous rows")
    if torch.is_grad_enabled() and logits.requires_grad:
        rest = []
        weights = _RouteWeights.apply(logits, int(top_k), bool(renormalize), rest)
        return weights, *rest
    return _run_route(logits, None, shape[1], int(top_k), bool(renormalize))


def moe_sort(experts: torch.Tensor, num_experts: int) -> ExpertOrder:
    """The sort of given expert choices int32 ``[tokens, top_k]``; ids outside
    ``[0, num_experts)`` mean no expert."""
    if experts.dim() != 2 or experts.dtype != torch.int32 or experts.device.type != "cuda" or not experts.is_contiguous():
        raise ValueError("experts must be a contiguous int32 [tokens, top_k] CUDA tensor")
    if not 1 <= num_experts <= 512 or not 1 <= experts.shape[1] <= 32:
        raise ValueError("between 1 and 512 experts and 1 and 32 choices are supported")
    return _run_route(None, experts, int(num_experts), experts.shape[1], False)[2]


def _check_order(order, dev):
    """(tokens, top_k, experts) of an order on `dev`."""
    position, source, offsets = order
    for name, t in (("position", position), ("source", source), ("offsets", offsets)):
        if t.dtype != torch.int32 or t.device != dev or not t.is_contiguous():
            raise ValueError(f"order.{name} must be contiguous int32 on the rows' device")
    shape, count = position.shape, offsets.shape
    if len(shape) != 2 or source.shape != (shape[0] * shape[1],) or len(count) != 1 or count[0] < 1:
        raise ValueError("order must be what moe_route or moe_sort returned")
    if not 1 <= shape[1] <= 32:
        raise ValueError("between 1 and 32 choices are supported")
    return shape[0], shape[1], count[0] - 1


def _check_rows(name, t, rows, like=None):
    """(pointer, row stride) of a [rows, width] tensor; `like`: one whose width, type and device it has."""
    shape, dtype = t.shape, t.dtype
    if dtype not in _TYPES or len(shape) != 2 or not t.is_cuda:
        raise ValueError(f"{name} must be a 2-D CUDA tensor of float32, bfloat16 or float16")
    width = shape[1]
    if shape[0] != rows:
        raise ValueError(f"{name} has the wrong shape")
    if like is not None and (width != like.shape[1] or dtype != like.dtype or t.device != like.device):
        raise ValueError(f"{name} must have the rows' width, type and device")
    vec = 16 // t.element_size()
    if width == 0 or width % vec:
        raise ValueError(f"{name}: rows must be a positive multiple of 16 bytes")
    stride = t.stride()
    if rows and (stride[1] != 1 or (rows > 1 and (stride[0] % vec or stride[0] < width))):
        raise ValueError(f"{name}: rows must be contiguous and a multiple of 16 bytes apart")
    ptr = t.data_ptr()
    if ptr % 16:
        raise ValueError(f"{name} must be 16-byte aligned")
    return ptr, stride[0] if rows > 1 else width


def _permute(name, like, src, residual, weights, position, offsets, sizes, out, grad, grad_weights, status):
    """Calls a permute entry point; src, residual, out and grad are (pointer, row stride)."""
    tokens, top_k, experts = sizes
    _capi.call(name, _capi.AspireMoePermuteArgs(
        _TYPES[like.dtype], *src, *residual, None if weights is None else weights.data_ptr(), position.data_ptr(),
        offsets.data_ptr(), experts, top_k, tokens, like.shape[1], *out, *grad,
        None if grad_weights is None else grad_weights.data_ptr(),
        None if status is None else status.data_ptr()), like.device)


_NO = (None, 0)


def _run_dispatch(x, src, position, offsets, sizes, status):
    width = x.shape[1]
    out = torch.empty(sizes[0] * sizes[1], width, dtype=x.dtype, device=x.device)
    if sizes[0]:
        _permute("aspire_moe_dispatch", x, src, _NO, None, position, offsets, sizes, (out.data_ptr(), width), _NO, None,
                 status)
    return out


def _run_combine(rows, src, weights, position, offsets, sizes, residual, out, status):
    if out is None:
        width = rows.shape[1]
        out = torch.empty(sizes[0], width, dtype=rows.dtype, device=rows.device)
        to = (out.data_ptr(), width)
    else:
        to = _check_rows("out", out, sizes[0], rows)
    if sizes[0]:
        _permute("aspire_moe_combine", rows, src, residual, weights, position, offsets, sizes, to, _NO, None, status)
    return out


def _grad_rows(g):
    """A gradient in the layout the kernels take (autograd may hand over any strides), as (it, (pointer, row stride))."""
    stride, width = g.stride(), g.shape[1]
    if stride[1] != 1 or stride[0] * g.element_size() % 16 or stride[0] < width or g.data_ptr() % 16:
        g = g.contiguous()
        stride = g.stride()
    return g, (g.data_ptr(), stride[0] if g.shape[0] > 1 else width)


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, src, position, offsets, sizes, status):
        ctx.save_for_backward(position, offsets)
        ctx.sizes, ctx.status = sizes, status
        return _run_dispatch(x, src, position, offsets, sizes, status)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        position, offsets = ctx.saved_tensors
        g, src = _grad_rows(grad)
        return (_run_combine(g, src, None, position, offsets, ctx.sizes, _NO, None, ctx.status),
                None, None, None, None, None)


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, residual, src, res, position, offsets, sizes, status):
        ctx.save_for_backward(rows, weights, position, offsets)
        ctx.src, ctx.sizes, ctx.status = src, sizes, status
        return _run_combine(rows, src, weights, position, offsets, sizes, res, None, status)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        rows, weights, position, offsets = ctx.saved_tensors
        need_rows, need_weights, need_residual = ctx.needs_input_grad[:3]
        d_rows = d_weights = None
        if need_rows or need_weights:
            to = _NO
            if need_rows:
                d_rows = torch.empty(rows.shape, dtype=rows.dtype, device=rows.device)
                to = (d_rows.data_ptr(), rows.shape[1])
            if need_weights:
                d_weights = torch.empty(weights.shape, dtype=torch.float32, device=rows.device)
            if ctx.sizes[0]:
                g, src = _grad_rows(grad)
                _permute("aspire_moe_combine_grad", rows, ctx.src, _NO, weights, position, offsets, ctx.sizes, to, src,
                         d_weights, ctx.status)
        return d_rows, d_weights, grad if need_residual else None, None, None, None, None, None, None


def moe_dispatch(x: torch.Tensor, order: ExpertOrder, *, status: torch.Tensor | None = None) -> torch.Tensor:
    """The tokens' rows sorted by expert: ``x [tokens, width]`` ->
    ``[tokens * top_k, width]``; rows past the last expert's are zero (C ABI
    ``aspire_moe_dispatch``)."""
    sizes = _check_order(order, x.device)
    src = _check_rows("x", x, sizes[0])
    if torch.is_grad_enabled() and x.requires_grad:
        return _Dispatch.apply(x, src, order[0], order[2], sizes, status)
    return _run_dispatch(x, src, order[0], order[2], sizes, status)


def moe_combine(rows: torch.Tensor, weights: torch.Tensor, order: ExpertOrder, *,
                residual: torch.Tensor | None = None, out: torch.Tensor | None = None,
                status: torch.Tensor | None = None) -> torch.Tensor:
    """``y[t] = sum_j weights[t, j] * rows[order.position[t, j]]``
    (``+ residual[t]``), summed in fp32 (C ABI ``aspire_moe_combine``).  ``out``
    may be ``residual`` itself; it takes no part in a gradient."""
    sizes = _check_order(order, rows.device)
    src = _check_rows("rows", rows, sizes[0] * sizes[1])
    if (weights.dtype != torch.float32 or weights.shape != sizes[:2] or weights.device != rows.device
            or not weights.is_contiguous()):
        raise ValueError("weights must be contiguous float32 [tokens, top_k] on the rows' device")
    res = _NO if residual is None else _check_rows("residual", residual, sizes[0], rows)
    if torch.is_grad_enabled() and (rows.requires_grad or weights.requires_grad
                                    or (residual is not None and residual.requires_grad)):
        if out is not None:
            raise ValueError("out cannot be given where a gradient is wanted")
        return _Combine.apply(rows, weights, residual, src, res, order[0], order[2], sizes, status)
    return _run_combine(rows, src, weights, order[0], order[2], sizes, res, out, status)
