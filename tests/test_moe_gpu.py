"""GPU tests of routing, dispatch and combine against their definitions in 64
bits, and of their gradients against the formulas and against differences."""

import pytest
import torch

from aspire_b200 import moe, quant
from ffn_reference import U, check, choose, product, random_w4, sort_slots

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
NINF = float("-inf")


def _randn(*shape, seed, dtype=torch.float32):
    g = torch.Generator(device="cpu")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype)


def _softmax(logits, chosen, renormalize):
    """Weights in 64 bits, from the definition."""
    x = logits.double().cpu()
    x = torch.where(torch.isnan(x), NINF, x)
    live = chosen >= 0
    v = torch.where(live, x.gather(1, chosen.clamp(min=0).long()), NINF)
    m = x.amax(1, keepdim=True)
    m = torch.where(m == NINF, 0.0, m)
    e = torch.where(live, (v - m).exp(), 0.0)
    total = e.sum(1, keepdim=True) if renormalize else (x - m).exp().sum(1, keepdim=True)
    return torch.where(live, e / torch.where(total > 0, total, 1.0), 0.0)


def _assert_order(order, chosen, experts):
    p, s, o = sort_slots(chosen, experts)
    assert torch.equal(order.position.cpu(), p)
    assert torch.equal(order.source.cpu(), s)
    assert torch.equal(order.offsets.cpu(), o)


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("tokens,experts,top_k", [
    (1, 1, 1), (1, 512, 32), (3, 7, 7), (72, 128, 8), (64, 60, 6), (128, 33, 8), (129, 128, 8), (1000, 160, 3),
    (1025, 256, 1), (2500, 512, 5), (700, 512, 32)])
def test_route(cuda_device, tokens, experts, top_k, renormalize):
    logits = _randn(tokens, experts, seed=tokens + experts)
    if tokens > 2:
        logits[1] = NINF                       # a padding row
        logits[2, : experts - 1] = NINF        # one expert left
    w, e, order = moe.moe_route(logits.to(cuda_device), top_k, renormalize=renormalize)
    chosen = choose(logits, top_k)
    assert torch.equal(e.cpu(), chosen)
    ref = _softmax(logits, chosen, renormalize)
    # Exponentials (2 ulp), a sum of at most 512 terms, a quotient.
    check(w, ref, ref * (512 * 2.0 ** -24 + 8 * 2.0 ** -24) + 1e-37)
    _assert_order(order, chosen, experts)


@pytest.mark.parametrize("dtype", TYPES)
def test_route_ties_nan_and_infinities(cuda_device, dtype):
    rows = [[1.0] * 40, [0.0, -0.0] * 20, [NINF] * 40, [float("nan")] * 40, [float("inf"), 1.0] + [float("inf")] * 38,
            [-3.0] * 39 + [2.0], [float("nan"), 5.0] + [NINF] * 38, [-6e4] * 20 + [6e4] * 20]
    logits = torch.tensor(rows).to(dtype)
    for renormalize in (True, False):
        w, e, order = moe.moe_route(logits.to(cuda_device), 4, renormalize=renormalize)
        chosen = choose(logits, 4)
        assert torch.equal(e.cpu(), chosen)
        _assert_order(order, chosen, 40)
        w = w.cpu()
        assert bool(torch.isfinite(w).all())
        assert bool((w[2] == 0).all()) and bool((w[3] == 0).all())
        assert w[6].tolist() == [1.0, 0.0, 0.0, 0.0]
        assert torch.allclose(w[0], torch.full((4,), 0.25 if renormalize else 1 / 40))
        assert torch.allclose(w[4], torch.full((4,), 0.25 if renormalize else 1 / 39))


@pytest.mark.parametrize("tokens,top_k,experts", [(1, 1, 4), (50, 3, 9), (400, 5, 512), (3000, 2, 17)])
def test_sort_of_given_choices(cuda_device, tokens, top_k, experts):
    g = torch.Generator(device="cpu")
    g.manual_seed(tokens)
    chosen = torch.randint(-2, experts + 2, (tokens, top_k), generator=g).to(torch.int32)
    _assert_order(moe.moe_sort(chosen.to(cuda_device), experts), chosen, experts)


def test_no_tokens(cuda_device):
    w, e, order = moe.moe_route(torch.empty(0, 8, device=cuda_device), 2)
    assert w.shape == (0, 2) and order.offsets.tolist() == [0] * 9
    rows = moe.moe_dispatch(torch.empty(0, 64, device=cuda_device), order)
    assert rows.shape == (0, 64)
    assert moe.moe_combine(rows, w, order).shape == (0, 64)


def _order(tokens, experts, top_k, device, seed, drop=0.2):
    g = torch.Generator(device="cpu")
    g.manual_seed(seed)
    chosen = torch.rand(tokens, experts, generator=g).argsort(1)[:, :top_k].to(torch.int32)
    chosen[torch.rand(tokens, top_k, generator=g) < drop] = -1
    if tokens > 1:
        chosen[1] = -1
    return moe.moe_sort(chosen.to(device), experts), chosen


CASES = [(1, 8, 1, 8), (5, 4, 4, 264), (64, 16, 8, 2048), (300, 60, 6, 1032), (17, 40, 32, 4096)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,experts,top_k,width", CASES)
def test_dispatch_and_gradient(cuda_device, tokens, experts, top_k, width, dtype):
    order, chosen = _order(tokens, experts, top_k, cuda_device, tokens)
    x = _randn(tokens, width, seed=1, dtype=dtype).to(cuda_device).requires_grad_()
    y = moe.moe_dispatch(x, order)
    position, source, offsets = sort_slots(chosen, experts)
    n = int(offsets[-1])
    want = torch.zeros(tokens * top_k, width, dtype=dtype)
    want[:n] = x.detach().cpu()[source[:n].long() // top_k]
    assert torch.equal(y.detach().cpu(), want)
    grad = _randn(tokens * top_k, width, seed=2, dtype=dtype).to(cuda_device)
    grad[n:] = float("nan")  # rows of no token take no part
    (gx,) = torch.autograd.grad(y, x, grad)
    rows = torch.where((position >= 0)[..., None], grad.double().cpu()[position.clamp(min=0).long()], 0.0)
    ref, mag = rows.sum(1), rows.abs().sum(1)
    check(gx, ref, ref.abs() * U[dtype] + mag * top_k * 2.0 ** -24 + 1e-7 * (dtype == torch.float16))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,experts,top_k,width", CASES)
def test_combine_and_gradients(cuda_device, tokens, experts, top_k, width, dtype):
    order, chosen = _order(tokens, experts, top_k, cuda_device, tokens)
    position, source, offsets = sort_slots(chosen, experts)
    n = int(offsets[-1])
    rows = _randn(tokens * top_k, width, seed=3, dtype=dtype).to(cuda_device)
    rows[n:] = float("nan")
    rows.requires_grad_()
    weights = _randn(tokens, top_k, seed=4).to(cuda_device).requires_grad_()
    res = _randn(tokens, width, seed=5, dtype=dtype).to(cuda_device).requires_grad_()
    live = (position >= 0)[..., None]
    r = torch.where(live, rows.detach().double().cpu()[position.clamp(min=0).long()], 0.0)
    w = weights.detach().double().cpu()
    tiny = 1e-7 * (dtype == torch.float16)
    for residual in (None, res):
        y = moe.moe_combine(rows, weights, order, residual=residual)
        terms = r * w[..., None]
        ref, mag = terms.sum(1), terms.abs().sum(1)
        if residual is not None:
            ref, mag = ref + res.detach().double().cpu(), mag + res.detach().double().cpu().abs()
        check(y.detach(), ref, ref.abs() * U[dtype] + mag * (top_k + 2) * 2.0 ** -24 + tiny)
    grad = _randn(tokens, width, seed=6, dtype=dtype).to(cuda_device)
    gr, gw, gres = torch.autograd.grad(y, (rows, weights, res), grad)
    assert torch.equal(gres, grad)
    g = grad.double().cpu()
    at = source[:n].long()
    ref = torch.zeros(tokens * top_k, width, dtype=torch.float64)
    ref[:n] = g[at // top_k] * w.reshape(-1)[at][:, None]
    check(gr, ref, ref.abs() * (U[dtype] + 2.0 ** -23) + tiny)
    dots, mags = (r * g[:, None]).sum(2), (r * g[:, None]).abs().sum(2)
    check(gw, dots, mags * width * 2.0 ** -24)


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("tokens,experts,top_k", [(1, 4, 2), (40, 33, 5), (300, 128, 8), (9, 512, 32)])
@pytest.mark.parametrize("dtype", TYPES)
def test_route_gradient(cuda_device, tokens, experts, top_k, renormalize, dtype):
    logits = _randn(tokens, experts, seed=7, dtype=dtype)
    if tokens > 2:
        logits[1] = NINF
        logits[2, 1:] = NINF
    x = logits.to(cuda_device).requires_grad_()
    w, e, _ = moe.moe_route(x, top_k, renormalize=renormalize)
    grad = _randn(tokens, top_k, seed=8).to(cuda_device)
    (gx,) = torch.autograd.grad(w, x, grad)
    chosen = choose(logits, top_k)
    p = _softmax(logits, chosen, renormalize)
    g = torch.where(chosen >= 0, grad.double().cpu(), 0.0)
    inner = (p * g).sum(1, keepdim=True)
    ref = torch.zeros(tokens, experts, dtype=torch.float64)
    mag = torch.zeros_like(ref)
    if not renormalize:
        ld = logits.double()
        m = torch.where(ld.amax(1, keepdim=True) == NINF, 0.0, ld.amax(1, keepdim=True))
        full = (ld - m).exp()
        full = full / full.sum(1, keepdim=True).clamp(min=1e-300)
        ref -= full * inner
        mag += full * (p * g).abs().sum(1, keepdim=True)
    at = chosen.clamp(min=0).long()
    own = p * (g - inner if renormalize else g)
    ref.scatter_add_(1, at, own)
    mag.scatter_add_(1, at, (p * g).abs() + p * (p * g).abs().sum(1, keepdim=True))
    check(gx, ref, ref.abs() * U[dtype] + mag * 1100 * 2.0 ** -24 + 1e-7 * (dtype == torch.float16) + 1e-37)


def test_route_gradient_by_differences(cuda_device):
    torch.manual_seed(3)
    logits = torch.randn(6, 12, device=cuda_device)
    grad = torch.randn(6, 3, device=cuda_device)
    for renormalize in (True, False):
        x = logits.clone().requires_grad_()
        w, e, _ = moe.moe_route(x, 3, renormalize=renormalize)
        (gx,) = torch.autograd.grad(w, x, grad)

        def f(l):
            v = l.double().gather(1, e.long())
            p = torch.softmax(v, 1) if renormalize else torch.softmax(l.double(), 1).gather(1, e.long())
            return (p * grad.double()).sum()
        h = 1e-4
        for t, i in [(0, 0), (1, 5), (2, int(e[2, 0])), (3, int(e[3, 2])), (5, int(e[5, 1]))]:
            up, down = logits.double().clone(), logits.double().clone()
            up[t, i] += h
            down[t, i] -= h
            # The second difference of the softmax is below 1; fp32 gradients are good to 1e-6.
            assert abs(((f(up) - f(down)) / (2 * h)).item() - gx[t, i].item()) <= 1e-6 + h * h * 10


def test_layer_of_4_bit_experts_in_a_graph(cuda_device):
    """Routing, dispatch, gated and plain expert products and the combine, as a
    decode step runs them, captured once and replayed on other tokens."""
    T, D, I, E, K = 13, 256, 192, 10, 3
    gu = random_w4((E, 2 * I), D, 64, False, torch.bfloat16, cuda_device, seed=1, scale=0.02)
    dn = random_w4((E, D), I, 32, True, torch.bfloat16, cuda_device, seed=2, scale=0.02)
    x = torch.zeros(T, D, dtype=torch.bfloat16, device=cuda_device)
    logits = torch.zeros(T, E, device=cuda_device)

    def layer():
        weights, experts, order = moe.moe_route(logits, K)
        rows = moe.moe_dispatch(x, order)
        h = quant.w4_expert_swiglu(rows, order.offsets, *gu[:3])
        y = quant.w4_expert_linear(h, order.offsets, *dn[:3])
        return moe.moe_combine(y, weights, order, residual=x), weights, experts, order, h, y
    layer()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, weights, experts, order, h, y = layer()
    for seed in (1, 2):
        x.copy_(_randn(T, D, seed=seed, dtype=torch.bfloat16))
        logits.copy_(_randn(T, E, seed=seed + 10))
        logits[4] = NINF
        g.replay()
        chosen = choose(logits, K)
        assert torch.equal(experts.cpu(), chosen)
        pos, src, off = sort_slots(chosen, E)
        n = int(off[-1])
        xs = x.cpu()[src[:n].long() // K]
        for e in range(E):
            a, b = int(off[e]), int(off[e + 1])
            ref, bound = product(xs[a:b], gu[3][e], swiglu=True, rows=T * K)
            check(h[a:b], ref, bound)
            ref, bound = product(h[a:b].cpu(), dn[3][e], rows=T * K)
            check(y[a:b], ref, bound)
        terms = torch.where((pos >= 0)[..., None], y.double().cpu()[pos.clamp(min=0).long()], 0.0)
        terms = terms * weights.double().cpu()[..., None]
        ref = terms.sum(1) + x.double().cpu()
        check(out, ref, ref.abs() * U[torch.bfloat16] + (terms.abs().sum(1) + x.double().cpu().abs()) * 8 * 2.0 ** -24)
        assert torch.equal(out[4], x[4])  # no expert: the residual alone


def test_bad_positions_are_reported(cuda_device):
    order, _ = _order(6, 4, 2, cuda_device, 1, drop=0.0)
    order = moe.ExpertOrder(order.position.clone(), order.source, order.offsets)
    order.position[0, 0] = 12
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    x = _randn(6, 64, seed=1).to(cuda_device)
    moe.moe_dispatch(x, order, status=status)
    assert int(status) & 4
    status.zero_()
    moe.moe_combine(torch.zeros(12, 64, device=cuda_device), torch.zeros(6, 2, device=cuda_device), order, status=status)
    assert int(status) & 4


def test_refusals(cuda_device):
    order, _ = _order(6, 4, 2, cuda_device, 1)
    x = _randn(6, 64, seed=1).to(cuda_device)
    rows, w = torch.zeros(12, 64, device=cuda_device), torch.zeros(6, 2, device=cuda_device)
    for call in (
        lambda: moe.moe_route(x.double(), 2), lambda: moe.moe_route(x, 0), lambda: moe.moe_route(x, 33),
        lambda: moe.moe_route(x[:, :3], 4), lambda: moe.moe_route(x.cpu(), 2), lambda: moe.moe_route(x.t(), 2),
        lambda: moe.moe_route(torch.zeros(2, 513, device=cuda_device), 2),
        lambda: moe.moe_sort(torch.zeros(2, 2, device=cuda_device), 4),
        lambda: moe.moe_dispatch(x[:5], order), lambda: moe.moe_dispatch(x[:, :63], order),
        lambda: moe.moe_dispatch(x.int(), order), lambda: moe.moe_combine(rows, w.half(), order),
        lambda: moe.moe_combine(rows[:10], w, order), lambda: moe.moe_combine(rows, w[:, :1], order),
        lambda: moe.moe_combine(rows, w, order, residual=x.half()),
        lambda: moe.moe_combine(rows, w.requires_grad_(), order, out=x),
    ):
        with pytest.raises(ValueError):
            call()


def test_gradients_of_any_layout(cuda_device):
    # Autograd hands over whatever the consumer made: broadcast, transposed, off a 16-byte boundary.
    tokens, experts, top_k, width = 5, 4, 2, 64
    order, _ = _order(tokens, experts, top_k, cuda_device, 3)
    x = _randn(tokens, width, seed=1).to(cuda_device).requires_grad_()
    rows = _randn(tokens * top_k, width, seed=2).to(cuda_device).requires_grad_()
    weights = _randn(tokens, top_k, seed=3).to(cuda_device).requires_grad_()
    for n, y, wrt in ((tokens * top_k, moe.moe_dispatch(x, order), (x,)),
                      (tokens, moe.moe_combine(rows, weights, order), (rows, weights))):
        off = torch.empty(n * width + 1, device=cuda_device)[1:].view(n, width)
        off.copy_(_randn(n, width, seed=4))
        for g in (off, _randn(width, n, seed=5).to(cuda_device).t(), torch.ones(1, 1, device=cuda_device).expand(n, width)):
            got = torch.autograd.grad(y, wrt, g, retain_graph=True)
            want = torch.autograd.grad(y, wrt, torch.empty(n, width, device=cuda_device).copy_(g), retain_graph=True)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
