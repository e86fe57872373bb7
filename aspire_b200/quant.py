"""Products with 4-bit weights and group scales (C ABI ``aspire_w4_linear``).

A decode step of the engine reads every weight matrix for a few tokens per row
(one when drafting, the drafts plus one when verifying), so its products are
bound by the weights' bytes; 4-bit weights are a quarter of the bf16 ones.
The same calls take a prefill chunk.

A matrix ``[n, k]`` is three tensors (:class:`W4Weight`):

* ``codes`` int32 ``[n, k / 8]``: a word holds eight consecutive weights,
  weight ``8w + 2i`` in bits ``4i..4i+3`` and weight ``8w + 2i + 1`` in bits
  ``16+4i..19+4i``;
* ``scales`` ``[n, k / group]`` in the type of the activations (bf16, fp16);
* ``zeros`` uint8 ``[n, k / group]`` (0..15), or ``None`` for 8 everywhere.

Weight ``(r, j)`` is ``(q - zero) * scale``.  ``group`` is 32, 64 or a multiple
of 128.  The experts of a sparse layer are one such matrix each, stacked in a
leading dimension.  The products have no gradient, of the weights or of ``x``:
with gradients enabled they refuse operands that require one.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _capi

_TYPES = (torch.bfloat16, torch.float16)
_NIBBLE = (0, 16, 4, 20, 8, 24, 12, 28)  # bit of each of a word's eight weights


@dataclass
class W4Weight:
    """A 4-bit matrix, or one per expert (leading dimension)."""

    codes: torch.Tensor
    scales: torch.Tensor
    zeros: torch.Tensor | None = None

    @property
    def group(self) -> int:
        return self.codes.shape[-1] * 8 // self.scales.shape[-1]


def _check_group(k: int, group: int) -> None:
    if group not in (32, 64) and (group <= 0 or group % 128):
        raise ValueError("group must be 32, 64 or a multiple of 128")
    if k % group:
        raise ValueError("k must be a multiple of group")


def quantize_w4(weight: torch.Tensor, group: int = 128, symmetric: bool = True) -> W4Weight:
    """Rounds ``weight`` ``[..., n, k]`` (bf16 or fp16) to 4 bits, group by
    group: symmetric (codes around 8, the largest magnitude at 8 steps) or with
    a zero point (the group's range, zero included, over 15 steps).  Codes are
    chosen against the scale as it is stored."""
    if weight.dtype not in _TYPES:
        raise ValueError("weight must be bfloat16 or float16")
    if weight.dim() < 2:
        raise ValueError("weight must be [..., n, k]")
    _check_group(weight.shape[-1], group)
    w = weight.float().unflatten(-1, (-1, group))
    tiny = torch.finfo(weight.dtype).tiny
    if symmetric:
        peak = w.gather(-1, w.abs().argmax(-1, keepdim=True))[..., 0]
        scales = (peak / -8).to(weight.dtype)
        scales = torch.where(scales.abs() < tiny, torch.full_like(scales, tiny), scales)
        z = torch.full_like(peak, 8.0)
        zeros = None
    else:
        lo, hi = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
        scales = ((hi - lo) / 15).clamp(min=tiny).to(weight.dtype)
        z = (-lo / scales.float()).round().clamp(0, 15)
        zeros = z.to(torch.uint8)
    q = (w / scales.float()[..., None] + z[..., None]).round().clamp(0, 15).to(torch.int32).flatten(-2)
    words = torch.zeros(*q.shape[:-1], q.shape[-1] // 8, dtype=torch.int32, device=q.device)
    for i, bit in enumerate(_NIBBLE):
        words |= q[..., i::8] << bit
    return W4Weight(words, scales, zeros)


def dequantize_w4(w: W4Weight) -> torch.Tensor:
    """The weights ``[..., n, k]`` in fp32."""
    shift = torch.tensor(_NIBBLE, device=w.codes.device, dtype=torch.int32)
    q = ((w.codes[..., None] >> shift) & 15).flatten(-2).float().unflatten(-1, (-1, w.group))
    z = 8.0 if w.zeros is None else w.zeros.float()[..., None]
    return ((q - z) * w.scales.float()[..., None]).flatten(-2)


def w4_linear(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None, *,
              residual: torch.Tensor | None = None, out: torch.Tensor | None = None,
              status: torch.Tensor | None = None) -> torch.Tensor:
    """``x [rows, k] @ W^T`` (``+ residual``) -> ``[rows, n]``, for one token up
    to a prefill chunk.  ``out`` may be ``residual`` itself; otherwise it must not
    overlap what the call reads."""
    return _capi.ops().w4(x, codes, scales, zeros, residual, out, False, None, status)


def w4_swiglu(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None, *,
              out: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """``silu(x G^T) * (x U^T)`` -> ``[rows, n]`` with the matrix's rows
    ``[0, n)`` the gate's and ``[n, 2n)`` the up product's."""
    return _capi.ops().w4(x, codes, scales, zeros, None, out, True, None, status)


def w4_expert_linear(x: torch.Tensor, offsets: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor,
                     zeros: torch.Tensor | None = None, *, out: torch.Tensor | None = None,
                     status: torch.Tensor | None = None) -> torch.Tensor:
    """Every row's product with its expert's matrix: rows
    ``offsets[e] .. offsets[e + 1]`` of ``x`` (sorted by expert, as
    :func:`aspire_b200.moe.moe_dispatch` leaves them) use matrix ``e``; rows
    before the first expert's and past the last one's give zero, so that the
    offsets may be those of a share of the experts."""
    return _capi.ops().w4(x, codes, scales, zeros, None, out, False, offsets, status)


def w4_expert_swiglu(x: torch.Tensor, offsets: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor,
                     zeros: torch.Tensor | None = None, *, out: torch.Tensor | None = None,
                     status: torch.Tensor | None = None) -> torch.Tensor:
    """The gated form of :func:`w4_expert_linear` (each expert's matrix holds
    its gate rows, then its up rows)."""
    return _capi.ops().w4(x, codes, scales, zeros, None, out, True, offsets, status)
