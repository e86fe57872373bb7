"""64-bit definitions of the feed-forward operators for their tests, and the
error bounds those follow from.

Bounds: a product's output is rounded once (half a unit in the last place, u =
2^-8 bf16 or 2^-11 fp16 relative); its sum runs in fp32, where each of the k
additions and roundings loses at most 2^-22 of the sum of magnitudes (the
matrix instructions may truncate); with more than 16 rows the weights are
rounded to the activations' type first (u of each weight's magnitude).
"""

from __future__ import annotations

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
BITS = [0, 16, 4, 20, 8, 24, 12, 28]


def random_w4(shape, k, group, zeros, dtype, device, seed, scale=0.01):
    """Random codes over all 16 values, positive and negative scales."""
    g = torch.Generator(device="cpu")
    g.manual_seed(seed)
    q = torch.randint(0, 16, (*shape, k), generator=g)
    words = torch.zeros(*shape, k // 8, dtype=torch.int64)
    for i, bit in enumerate(BITS):
        words |= q[..., i::8] << bit
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
    s = ((torch.rand(*shape, k // group, generator=g) + 0.25) * scale
         * torch.where(torch.rand(*shape, k // group, generator=g) < 0.5, -1.0, 1.0)).to(dtype)
    z = torch.randint(0, 16, (*shape, k // group), generator=g).to(torch.uint8) if zeros else None
    w = (q.double() - (8.0 if z is None else z.double().repeat_interleave(group, -1)))
    w = w * s.double().repeat_interleave(group, -1)
    dev = lambda t: None if t is None else t.to(device)  # noqa: E731
    return dev(words), dev(s), dev(z), w


def product(x, w, residual=None, swiglu=False, rows=None):
    """(reference, bound) of x [rows, k] with w [n, k], both float64 on the CPU;
    `rows` is the call's row count (it decides whether weights are rounded)."""
    dtype = x.dtype
    u = U[dtype]
    xd = x.double().cpu()
    y = xd @ w.t()
    mag = xd.abs() @ w.abs().t()
    k = w.shape[1]
    err = mag * (k * 2.0 ** -22 + (u if (rows if rows is not None else x.shape[0]) > 16 else 0.0))
    if swiglu:
        n = w.shape[0] // 2
        a, b, ea, eb = y[:, :n], y[:, n:], err[:, :n], err[:, n:]
        s = a * torch.sigmoid(a)
        y = s * b
        # |silu'| <= 1.1; the fast exponential loses 2^-21 (1 + |a|) relative.
        err = 1.1 * ea * (b.abs() + eb) + s.abs() * eb + y.abs() * (1 + a.abs()) * 2.0 ** -20
    if residual is not None:
        y = y + residual.double().cpu()
        err = err + y.abs() * 2.0 ** -23
    # Subnormal outputs are rounded to the type's smallest step.
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return y, err * (1 + u) + y.abs() * u + tiny


def check(got, ref, bound, what=""):
    d = (got.double().cpu() - ref).abs()
    bad = ~(d <= bound)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} out, worst {(d / bound.clamp(min=1e-300)).max():.3g} x bound"


def choose(logits, top_k):
    """Chosen experts: by value, then by index; NaN and -inf never."""
    tokens, experts = logits.shape
    out = torch.full((tokens, top_k), -1, dtype=torch.int32)
    rows = logits.double().cpu().tolist()
    for t in range(tokens):
        order = sorted((e for e in range(experts) if rows[t][e] == rows[t][e] and rows[t][e] > float("-inf")),
                       key=lambda e: (-rows[t][e], e))[:top_k]
        out[t, :len(order)] = torch.tensor(order, dtype=torch.int32)
    return out


def sort_slots(chosen, experts):
    """position, source, offsets by the definition."""
    flat = chosen.reshape(-1).tolist()
    order = sorted((i for i, e in enumerate(flat) if 0 <= e < experts), key=lambda i: (flat[i], i))
    position = torch.full((len(flat),), -1, dtype=torch.int32)
    source = torch.full((len(flat),), -1, dtype=torch.int32)
    for p, i in enumerate(order):
        position[i] = p
        source[p] = i
    counts = [0] * experts
    for i in order:
        counts[flat[i]] += 1
    offsets = torch.tensor([0] + counts).cumsum(0).to(torch.int32)
    return position.view(chosen.shape), source, offsets
