"""GPU tests of the 4-bit products against their definition in 64 bits."""

import pytest
import torch

from aspire_b200 import quant
from ffn_reference import check, product, random_w4

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _x(rows, k, dtype, device, seed):
    g = torch.Generator(device="cpu")
    g.manual_seed(seed)
    return torch.randn(rows, k, generator=g).to(dtype).to(device)


@pytest.mark.parametrize("rows", [1, 3, 8, 9, 16, 17, 32, 33, 64, 65, 129, 300])
@pytest.mark.parametrize("n,k,group,zeros,dtype", [
    (1, 32, 32, False, BF16),
    (130, 288, 32, True, BF16),
    (631, 832, 64, False, F16),
    (256, 2048, 128, False, BF16),
    (384, 768, 256, True, BF16),
    (77, 1920, 640, True, F16),
    (200, 5248, 64, True, BF16),
])
def test_linear(cuda_device, rows, n, k, group, zeros, dtype):
    codes, scales, z, w = random_w4((n,), k, group, zeros, dtype, cuda_device, seed=n + k)
    x = _x(rows, k, dtype, cuda_device, rows)
    res = _x(rows, n, dtype, cuda_device, rows + 1)
    ref, bound = product(x, w)
    check(quant.w4_linear(x, codes, scales, z), ref, bound, "plain")
    ref, bound = product(x, w, residual=res)
    check(quant.w4_linear(x, codes, scales, z, residual=res), ref, bound, "residual")


@pytest.mark.parametrize("rows", [1, 9, 31, 64, 200])
@pytest.mark.parametrize("n,k,group,zeros,dtype", [
    (1, 64, 64, False, BF16),
    (65, 544, 32, True, BF16),
    (391, 1152, 128, True, F16),
    (768, 2048, 128, False, BF16),
])
def test_swiglu(cuda_device, rows, n, k, group, zeros, dtype):
    codes, scales, z, w = random_w4((2 * n,), k, group, zeros, dtype, cuda_device, seed=n + k)
    x = _x(rows, k, dtype, cuda_device, rows)
    ref, bound = product(x, w, swiglu=True)
    check(quant.w4_swiglu(x, codes, scales, z), ref, bound)


@pytest.mark.parametrize("counts,tail", [
    ([0, 0, 5, 0, 1, 9, 0], 0),
    ([3], 0),
    ([0, 0, 0], 4),
    ([40, 1, 0, 33, 8, 0, 200], 11),
    ([1] * 70, 3),
])
@pytest.mark.parametrize("n,k,group,zeros,dtype,swiglu", [
    (72, 288, 32, True, BF16, False),
    (296, 640, 128, False, BF16, True),
    (130, 512, 64, True, F16, False),
])
def test_experts(cuda_device, counts, tail, n, k, group, zeros, dtype, swiglu):
    E = len(counts)
    r = 2 * n if swiglu else n
    codes, scales, z, w = random_w4((E, r), k, group, zeros, dtype, cuda_device, seed=E + n)
    rows = sum(counts) + tail
    x = _x(rows, k, dtype, cuda_device, 5)
    offsets = torch.tensor([0] + counts).cumsum(0).to(torch.int32).to(cuda_device)
    call = quant.w4_expert_swiglu if swiglu else quant.w4_expert_linear
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    y = call(x, offsets, codes, scales, z, out=torch.full((rows, n), float("nan"), dtype=dtype, device=cuda_device),
             status=status)
    at = 0
    for e, c in enumerate(counts):
        # The larger bound (rounded weights) where the call may take either path.
        ref, bound = product(x[at:at + c], w[e], swiglu=swiglu, rows=rows)
        check(y[at:at + c], ref, bound, f"expert {e}")
        at += c
    assert bool((y[at:] == 0).all())
    assert int(status) == 0


def test_experts_with_broken_offsets_stay_in_bounds(cuda_device):
    codes, scales, z, w = random_w4((3, 128), 128, 128, False, BF16, cuda_device, seed=1)
    x = _x(6, 128, BF16, cuda_device, 2)
    guard = torch.full((10, 128), 7.0, dtype=BF16, device=cuda_device)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    offsets = torch.tensor([0, 2, 99, 6], dtype=torch.int32, device=cuda_device)
    quant.w4_expert_linear(x, offsets, codes, scales, z, out=guard[2:8], status=status)
    assert int(status) & 4
    assert bool((guard[:2] == 7).all()) and bool((guard[8:] == 7).all())
    ref, bound = product(x[:2], w[0], rows=6)
    check(guard[2:4], ref, bound)


@pytest.mark.parametrize("rows", [2, 20, 70])
def test_strides_and_in_place_residual(cuda_device, rows):
    n, k, group = 136, 512, 64
    codes, scales, z, w = random_w4((n + 9,), k + 64, group, True, BF16, cuda_device, seed=3)
    x = _x(rows, k + 24, BF16, cuda_device, 4)[:, 8:8 + k]
    codes, scales, z = codes[4:4 + n, :k // 8], scales[4:4 + n, :k // group], z[4:4 + n, :k // group]
    buf = _x(rows, n + 3, BF16, cuda_device, 6)
    before = buf.clone()
    ref, bound = product(x, w[4:4 + n, :k], residual=before[:, 1:1 + n])
    view = buf[:, 1:1 + n]
    assert quant.w4_linear(x, codes, scales, z, residual=view, out=view) is view
    check(view, ref, bound)
    assert torch.equal(buf[:, :1], before[:, :1]) and torch.equal(buf[:, 1 + n:], before[:, 1 + n:])


@pytest.mark.parametrize("rows", [5, 40])
def test_nan_and_inf_stay_in_their_rows(cuda_device, rows):
    codes, scales, z, w = random_w4((160,), 320, 32, True, BF16, cuda_device, seed=8)
    x = _x(rows, 320, BF16, cuda_device, 9)
    x[1, 7] = float("nan")
    x[2, 300] = float("inf")
    y = quant.w4_linear(x, codes, scales, z)
    assert bool(torch.isnan(y[1]).all())
    live = (w[:, 300] != 0).to(cuda_device)
    assert bool(torch.isinf(y[2][live]).all())
    keep = [i for i in range(rows) if i not in (1, 2)]
    ref, bound = product(x[keep], w, rows=rows)
    check(y[keep], ref, bound)


@pytest.mark.parametrize("rows", [1, 12, 90])
def test_repeats_bit_by_bit_on_another_stream_and_in_a_graph(cuda_device, rows):
    codes, scales, z, w = random_w4((512,), 2048, 128, False, BF16, cuda_device, seed=11)
    x = _x(rows, 2048, BF16, cuda_device, 12)
    y = quant.w4_linear(x, codes, scales, z)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x2 = x * 1
        y2 = quant.w4_linear(x2, codes, scales, z)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, y2)
    out = torch.empty_like(y)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        quant.w4_linear(x2, codes, scales, z, out=out)
    x2.copy_(-x)
    g.replay()
    assert torch.equal(out, -y)


def test_no_rows(cuda_device):
    codes, scales, z, _ = random_w4((64,), 64, 32, True, BF16, cuda_device, seed=1)
    assert quant.w4_linear(torch.empty(0, 64, dtype=BF16, device=cuda_device), codes, scales, z).shape == (0, 64)


def test_refusals(cuda_device):
    codes, scales, z, _ = random_w4((64,), 256, 64, True, BF16, cuda_device, seed=1)
    x = _x(2, 256, BF16, cuda_device, 1)
    for bad in (dict(x=x.float()), dict(x=x.half()), dict(x=x[:, :128]), dict(codes=codes.long()),
                dict(scales=scales.half()), dict(scales=scales[:, :3]), dict(zeros=z.int()), dict(zeros=z[:, :1]),
                dict(x=x.cpu()), dict(x=x.t().contiguous().t()), dict(residual=x[:, :63]), dict(out=x[:, :64].float()),
                dict(x=_x(2, 260, BF16, cuda_device, 1)[:, 4:])):
        args = dict(x=x, codes=codes, scales=scales, zeros=z, **{})
        args.update(bad)
        with pytest.raises(ValueError):
            quant.w4_linear(args.pop("x"), args.pop("codes"), args.pop("scales"), args.pop("zeros"), **args)
    with pytest.raises(ValueError):
        quant.w4_swiglu(x, codes[:63], scales[:63], z[:63])
    with pytest.raises(ValueError):
        quant.w4_expert_linear(x, torch.zeros(3, dtype=torch.int32, device=cuda_device), codes[None], scales[None])


@pytest.mark.parametrize("symmetric", [True, False])
def test_quantized_weights_through_the_product(cuda_device, symmetric):
    g = torch.Generator(device="cpu")
    g.manual_seed(5)
    weight = (torch.randn(200, 512, generator=g) * 0.02).to(BF16)
    q = quant.quantize_w4(weight.to(cuda_device), 64, symmetric)
    w = quant.dequantize_w4(q).double().cpu()
    x = _x(4, 512, BF16, cuda_device, 6)
    ref, bound = product(x, w)
    check(quant.w4_linear(x, q.codes, q.scales, q.zeros), ref, bound)


@pytest.mark.parametrize("rows,n,k,group,zeros,dtype,swiglu", [
    (1500, 3000, 4096, 32, True, BF16, False),
    (1500, 3000, 4096, 32, True, F16, False),
    (700, 2048, 2048, 64, True, BF16, True),
    (48, 12000, 4096, 128, False, BF16, True),
    (16, 20000, 4096, 64, True, BF16, False),
])
def test_large_products_repeat_bit_by_bit(cuda_device, rows, n, k, group, zeros, dtype, swiglu):
    """Many tiles per CTA in a row: a stage that is released or read a moment
    too early shows in some of the runs."""
    codes, scales, z, w = random_w4((2 * n if swiglu else n,), k, group, zeros, dtype, cuda_device, seed=n)
    x = _x(rows, k, dtype, cuda_device, 3)
    call = quant.w4_swiglu if swiglu else quant.w4_linear
    first = call(x, codes, scales, z)
    for _ in range(15):
        assert torch.equal(call(x, codes, scales, z), first)
    some = list(range(0, rows, max(1, rows // 40)))  # every tile of tokens
    ref, bound = product(x[some], w, swiglu=swiglu, rows=rows)
    check(first[some], ref, bound)


@pytest.mark.parametrize("rows,n,k,expires", [(300, 2048, 1024, True), (40, 512, 4096, False)])
def test_expired_waits_are_reported_and_leave_the_device_usable(cuda_device, built_library, rows, n, k, expires):
    """With a wait limit of 1 ns the tcgen05 kernel stops at its first wait that
    a poll finds unfinished: it reports a timeout, and the next call gives the
    same result as before.  (In the second case, a cluster with few stages, a
    poll may outlast every wait; then the result has to be right.)"""
    codes, scales, z, w = random_w4((n,), k, 64, True, BF16, cuda_device, seed=2)
    x = _x(rows, k, BF16, cuda_device, 3)
    want = quant.w4_linear(x, codes, scales, z)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    built_library.aspire_set_wait_limit_ns(1)
    try:
        got = quant.w4_linear(x, codes, scales, z, status=status)
        torch.cuda.synchronize()
    finally:
        built_library.aspire_set_wait_limit_ns(0)
    timed_out = bool(int(status) & 8)
    assert timed_out or (not expires and torch.equal(got, want))
    assert torch.equal(quant.w4_linear(x, codes, scales, z), want)
