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

import ctypes
from typing import NamedTuple

import torch

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


def _call(name, args, dev):
    stream = torch.cuda.current_stream(dev).cuda_stream
    with torch.cuda.device(dev):
        rc = getattr(_capi.load_library(), name)(ctypes.byref(args), ctypes.c_void_p(stream))
    _capi.check(rc, name)


def _run_route(logits, experts, num_experts, top_k, renormalize):
    given = logits if logits is not None else experts
    tokens, dev = given.shape[0], given.device
    weights = None
    position = torch.empty(tokens, top_k, dtype=torch.int32, device=dev)
    source = torch.empty(tokens * top_k, dtype=torch.int32, device=dev)
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=dev)
    a = _capi.AspireMoeRouteArgs()
    if logits is not None:
        weights = torch.empty(tokens, top_k, dtype=torch.float32, device=dev)
        experts = torch.empty(tokens, top_k, dtype=torch.int32, device=dev)
        a.logits, a.logits_type = logits.data_ptr(), _TYPES[logits.dtype]
        a.logits_stride = logits.stride(0)
        a.weights = weights.data_ptr()
    a.tokens, a.num_experts, a.top_k, a.renormalize = tokens, num_experts, top_k, int(renormalize)
    a.experts, a.position = experts.data_ptr(), position.data_ptr()
    a.source, a.offsets = source.data_ptr(), offsets.data_ptr()
    need = _capi.load_library().aspire_moe_route_workspace(tokens, num_experts, top_k)
    if need:
        ws = torch.empty(need // 4, dtype=torch.int32, device=dev)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
    _call("aspire_moe_route", a, dev)
    return weights, experts, ExpertOrder(position, source, offsets)


class _RouteWeights(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_k, renormalize):
        weights, experts, order = _run_route(logits, None, logits.shape[1], top_k, renormalize)
        ctx.renormalize = renormalize
        ctx.logits_dtype, ctx.shape = logits.dtype, logits.shape
        ctx.save_for_backward(weights, experts, *([] if renormalize else [logits]))
        ctx.mark_non_differentiable(experts, *order)
        return (weights, experts, *order)

    @staticmethod
    def backward(ctx, grad_weights, *_):
        weights, experts, *rest = ctx.saved_tensors
        grad = torch.empty(ctx.shape, dtype=ctx.logits_dtype, device=weights.device)
        if grad.numel() == 0:
            return grad, None, None
        g = grad_weights.to(torch.float32).contiguous()
        a = _capi.AspireMoeRouteGradArgs()
        a.logits_type = _TYPES[ctx.logits_dtype]
        if rest:
            a.logits, a.logits_stride = rest[0].data_ptr(), rest[0].stride(0)
        a.weights, a.experts, a.grad_weights = weights.data_ptr(), experts.data_ptr(), g.data_ptr()
        a.tokens, a.num_experts = ctx.shape
        a.top_k, a.renormalize = weights.shape[1], int(ctx.renormalize)
        a.grad_logits = grad.data_ptr()
        _call("aspire_moe_route_grad", a, weights.device)
        return grad, None, None


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
    if logits.dim() != 2 or logits.dtype not in _TYPES or logits.device.type != "cuda":
        raise ValueError("logits must be a [tokens, experts] CUDA tensor of float32, bfloat16 or float16")
    if not 1 <= logits.shape[1] <= 512:
        raise ValueError("between 1 and 512 experts are supported")
    if not 1 <= top_k <= min(32, logits.shape[1]):
        raise ValueError("top_k must be between 1 and min(32, experts)")
    if logits.stride(1) != 1 and logits.shape[1] > 1 and logits.shape[0]:
        raise ValueError("logits need contiguous rows")
    if torch.is_grad_enabled() and logits.requires_grad:
        weights, experts, *order = _RouteWeights.apply(logits, int(top_k), bool(renormalize))
        return weights, experts, ExpertOrder(*order)
    return _run_route(logits, None, logits.shape[1], int(top_k), bool(renormalize))


def moe_sort(experts: torch.Tensor, num_experts: int) -> ExpertOrder:
    """The sort of given expert choices int32 ``[tokens, top_k]``; ids outside
    ``[0, num_experts)`` mean no expert."""
    if experts.dim() != 2 or experts.dtype != torch.int32 or experts.device.type != "cuda" or not experts.is_contiguous():
        raise ValueError("experts must be a contiguous int32 [tokens, top_k] CUDA tensor")
    if not 1 <= num_experts <= 512 or not 1 <= experts.shape[1] <= 32:
        raise ValueError("between 1 and 512 experts and 1 and 32 choices are supported")
    return _run_route(None, experts, int(num_experts), experts.shape[1], False)[2]


def _check_order(order, dev):
    position, source, offsets = order
    for name, t in (("position", position), ("source", source), ("offsets", offsets)):
        if t.dtype != torch.int32 or t.device != dev or not t.is_contiguous():
            raise ValueError(f"order.{name} must be contiguous int32 on the rows' device")
    if position.dim() != 2 or source.shape != (position.numel(),) or offsets.dim() != 1 or offsets.shape[0] < 1:
        raise ValueError("order must be what moe_route or moe_sort returned")
    if not 1 <= position.shape[1] <= 32:
        raise ValueError("between 1 and 32 choices are supported")


def _check_rows(name, t, rows, width=None):
    if t.dtype not in _TYPES or t.dim() != 2 or t.device.type != "cuda":
        raise ValueError(f"{name} must be a 2-D CUDA tensor of float32, bfloat16 or float16")
    if t.shape[0] != rows or (width is not None and t.shape[1] != width):
        raise ValueError(f"{name} has the wrong shape")
    vec = 16 // t.element_size()
    if t.shape[1] == 0 or t.shape[1] % vec:
        raise ValueError(f"{name}: rows must be a positive multiple of 16 bytes")
    if rows and (t.stride(1) != 1 or (rows > 1 and (t.stride(0) % vec or t.stride(0) < t.shape[1]))):
        raise ValueError(f"{name}: rows must be contiguous and a multiple of 16 bytes apart")
    if t.data_ptr() % 16:
        raise ValueError(f"{name} must be 16-byte aligned")


def _stride(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _permute_args(kind, order, width, status):
    a = _capi.AspireMoePermuteArgs()
    a.type, a.width = kind, width
    a.position, a.offsets = order[0].data_ptr(), order[2].data_ptr()
    a.tokens, a.top_k = order[0].shape
    a.num_experts = order[2].shape[0] - 1
    if status is not None:
        a.status = status.data_ptr()
    return a


def _run_dispatch(x, order, status):
    out = torch.empty(order[1].shape[0], x.shape[1], dtype=x.dtype, device=x.device)
    if out.numel():
        a = _permute_args(_TYPES[x.dtype], order, x.shape[1], status)
        a.in_, a.in_stride = x.data_ptr(), _stride(x)
        a.out, a.out_stride = out.data_ptr(), x.shape[1]
        _call("aspire_moe_dispatch", a, x.device)
    return out


def _run_combine(rows, weights, order, residual, out, status):
    if out is None:
        out = torch.empty(order[0].shape[0], rows.shape[1], dtype=rows.dtype, device=rows.device)
    if out.numel():
        a = _permute_args(_TYPES[rows.dtype], order, rows.shape[1], status)
        a.in_, a.in_stride = rows.data_ptr(), _stride(rows)
        a.out, a.out_stride = out.data_ptr(), _stride(out)
        if weights is not None:
            a.weights = weights.data_ptr()
        if residual is not None:
            a.residual, a.residual_stride = residual.data_ptr(), _stride(residual)
        _call("aspire_moe_combine", a, rows.device)
    return out


def _grad_rows(g):
    """A gradient in the layout the kernels take (autograd may hand over any strides)."""
    vec = 16 // g.element_size()
    ok = g.stride(1) == 1 and g.stride(0) % vec == 0 and g.stride(0) >= g.shape[1] and g.data_ptr() % 16 == 0
    return g if ok else g.contiguous()


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, position, source, offsets, status):
        ctx.save_for_backward(position, source, offsets)
        ctx.status = status
        return _run_dispatch(x, (position, source, offsets), status)

    @staticmethod
    def backward(ctx, grad):
        return _run_combine(_grad_rows(grad), None, ctx.saved_tensors, None, None, ctx.status), None, None, None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, position, source, offsets, residual, status):
        ctx.save_for_backward(rows, weights, position, source, offsets)
        ctx.status = status
        return _run_combine(rows, weights, (position, source, offsets), residual, None, status)

    @staticmethod
    def backward(ctx, grad):
        rows, weights, *order = ctx.saved_tensors
        need_rows, need_weights = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        d_rows = d_weights = None
        if (need_rows or need_weights) and grad.numel():
            g = _grad_rows(grad)
            a = _permute_args(_TYPES[rows.dtype], order, rows.shape[1], ctx.status)
            a.in_, a.in_stride = rows.data_ptr(), _stride(rows)
            a.weights = weights.data_ptr()
            a.grad, a.grad_stride = g.data_ptr(), _stride(g)
            if need_rows:
                d_rows = torch.empty(rows.shape, dtype=rows.dtype, device=rows.device)
                a.out, a.out_stride = d_rows.data_ptr(), rows.shape[1]
            if need_weights:
                d_weights = torch.empty_like(weights)
                a.grad_weights = d_weights.data_ptr()
            _call("aspire_moe_combine_grad", a, rows.device)
        elif need_rows or need_weights:
            d_rows = torch.zeros_like(rows) if need_rows else None
            d_weights = torch.zeros_like(weights) if need_weights else None
        return d_rows, d_weights, None, None, None, grad if ctx.needs_input_grad[5] else None, None


def moe_dispatch(x: torch.Tensor, order: ExpertOrder, *, status: torch.Tensor | None = None) -> torch.Tensor:
    """The tokens' rows sorted by expert: ``x [tokens, width]`` ->
    ``[tokens * top_k, width]``; rows past the last expert's are zero (C ABI
    ``aspire_moe_dispatch``)."""
    _check_rows("x", x, order[0].shape[0])
    _check_order(order, x.device)
    if torch.is_grad_enabled() and x.requires_grad:
        return _Dispatch.apply(x, *order, status)
    return _run_dispatch(x, order, status)


def moe_combine(rows: torch.Tensor, weights: torch.Tensor, order: ExpertOrder, *,
                residual: torch.Tensor | None = None, out: torch.Tensor | None = None,
                status: torch.Tensor | None = None) -> torch.Tensor:
    """``y[t] = sum_j weights[t, j] * rows[order.position[t, j]]``
    (``+ residual[t]``), summed in fp32 (C ABI ``aspire_moe_combine``).  ``out``
    may be ``residual`` itself; it takes no part in a gradient."""
    tokens = order[0].shape[0]
    _check_rows("rows", rows, order[0].numel())
    _check_order(order, rows.device)
    if weights.dtype != torch.float32 or weights.shape != order[0].shape or weights.device != rows.device:
        raise ValueError("weights must be float32 [tokens, top_k] on the rows' device")
    if not weights.is_contiguous():
        raise ValueError("weights must be contiguous")
    for name, t in (("residual", residual), ("out", out)):
        if t is not None:
            _check_rows(name, t, tokens, rows.shape[1])
            if t.dtype != rows.dtype or t.device != rows.device:
                raise ValueError(f"{name} must have the rows' type and device")
    needs = rows.requires_grad or weights.requires_grad or (residual is not None and residual.requires_grad)
    if torch.is_grad_enabled() and needs:
        if out is not None:
            raise ValueError("out cannot be given where a gradient is wanted")
        return _Combine.apply(rows, weights, *order, residual, status)
    return _run_combine(rows, weights, order, residual, out, status)
