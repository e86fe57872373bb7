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


class _RouteWeights(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_k, renormalize, rest):
        # Only the weights have a gradient; the integers go out by `rest`.
        weights, experts, *order = _capi.ops().route(logits, top_k, renormalize)
        rest += (experts, ExpertOrder(*order))
        ctx.how = logits.shape[1], _TYPES[logits.dtype], renormalize
        if renormalize:
            ctx.save_for_backward(weights, experts)
        else:
            ctx.save_for_backward(weights, experts, logits)
        return weights

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_weights):
        weights, experts, *rest = ctx.saved_tensors
        grad = _capi.ops().route_grad(grad_weights, weights, experts, rest[0] if rest else None, *ctx.how)
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
    if torch.is_grad_enabled() and logits.requires_grad:
        rest = []
        weights = _RouteWeights.apply(logits, top_k, bool(renormalize), rest)
        return weights, *rest
    weights, experts, *order = _capi.ops().route(logits, top_k, bool(renormalize))
    return weights, experts, ExpertOrder(*order)


def moe_sort(experts: torch.Tensor, num_experts: int) -> ExpertOrder:
    """The sort of given expert choices int32 ``[tokens, top_k]``; ids outside
    ``[0, num_experts)`` mean no expert."""
    return ExpertOrder(*_capi.ops().sort(experts, num_experts))


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, position, source, offsets, status):
        ctx.save_for_backward(position, source, offsets)
        ctx.status = status
        return _capi.ops().dispatch(x, position, source, offsets, status)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return _capi.ops().dispatch_grad(grad, *ctx.saved_tensors, ctx.status), None, None, None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, residual, position, source, offsets, status):
        ctx.save_for_backward(rows, weights, position, source, offsets)
        ctx.status = status
        return _capi.ops().combine(rows, weights, position, source, offsets, residual, None, status)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        need_rows, need_weights, need_residual = ctx.needs_input_grad[:3]
        d_rows = d_weights = None
        if need_rows or need_weights:
            d_rows, d_weights = _capi.ops().combine_grad(grad, *ctx.saved_tensors, need_rows, need_weights, ctx.status)
        return d_rows, d_weights, grad if need_residual else None, None, None, None, None


def moe_dispatch(x: torch.Tensor, order: ExpertOrder, *, status: torch.Tensor | None = None) -> torch.Tensor:
    """The tokens' rows sorted by expert: ``x [tokens, width]`` ->
    ``[tokens * top_k, width]``; rows past the last expert's are zero (C ABI
    ``aspire_moe_dispatch``)."""
    if torch.is_grad_enabled() and x.requires_grad:
        return _Dispatch.apply(x, *order, status)
    return _capi.ops().dispatch(x, *order, status)


def moe_combine(rows: torch.Tensor, weights: torch.Tensor, order: ExpertOrder, *,
                residual: torch.Tensor | None = None, out: torch.Tensor | None = None,
                status: torch.Tensor | None = None) -> torch.Tensor:
    """``y[t] = sum_j weights[t, j] * rows[order.position[t, j]]``
    (``+ residual[t]``), summed in fp32 (C ABI ``aspire_moe_combine``).  ``out``
    may be ``residual`` itself, otherwise it must not overlap what the call reads;
    it takes no part in a gradient."""
    if torch.is_grad_enabled() and (rows.requires_grad or weights.requires_grad
                                    or (residual is not None and residual.requires_grad)):
        if out is not None:
            raise ValueError("out cannot be given where a gradient is wanted")
        return _Combine.apply(rows, weights, residual, *order, status)
    return _capi.ops().combine(rows, weights, *order, residual, out, status)
