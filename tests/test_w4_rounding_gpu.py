"""GPU tests of what the 4-bit products round: nothing but the output up to 16
rows (8 per expert on average), and the weights, once, to the activations' type
above.  Also the experts' products with many tiles per CTA."""

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


# Short sums: the bound on fp32 additions, k 2^-22 of the magnitudes, is then far
# below what a rounding of the weights (2^-9 or 2^-12 of each) adds up to.
@pytest.mark.parametrize("k,group", [(128, 32), (256, 64), (128, 128)])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows", [1, 8, 16, 17, 64, 200])
def test_products_round_the_weights_above_16_rows_only(cuda_device, rows, dtype, k, group):
    n = 1000
    codes, scales, z, w = random_w4((n,), k, group, True, dtype, cuda_device, seed=rows + k)
    x = _x(rows, k, dtype, cuda_device, 1)
    y = quant.w4_linear(x, codes, scales, z)
    used, other = w, w.float().to(dtype).double()
    if rows > 16:
        used, other = other, used
    ref, bound = product(x, used, rows=1)
    check(y, ref, bound)
    if rows * n > 10000:  # (enough outputs near zero to tell the two apart)
        with pytest.raises(AssertionError):
            check(y, *product(x, other, rows=1))


@pytest.mark.parametrize("counts", [[1] * 70, [0, 30, 2, 0, 8, 0, 0, 16], [8] * 5, [9] * 5, [0, 0, 100, 3, 60]])
@pytest.mark.parametrize("k,group,zeros,dtype,swiglu", [
    (128, 32, True, BF16, False), (256, 128, False, BF16, True), (128, 64, True, F16, False)])
def test_experts_round_the_weights_above_8_rows_only(cuda_device, counts, k, group, zeros, dtype, swiglu):
    n, E, rows = 200, len(counts), sum(counts)
    codes, scales, z, w = random_w4((E, 2 * n if swiglu else n), k, group, zeros, dtype, cuda_device, seed=E)
    x = _x(rows, k, dtype, cuda_device, 2)
    offsets = torch.tensor([0] + counts).cumsum(0).to(torch.int32).to(cuda_device)
    y = (quant.w4_expert_swiglu if swiglu else quant.w4_expert_linear)(x, offsets, codes, scales, z)
    if -(-rows // E) > 8:
        w = w.float().to(dtype).double()
    at = 0
    for e, c in enumerate(counts):
        ref, bound = product(x[at:at + c], w[e], swiglu=swiglu, rows=1)
        check(y[at:at + c], ref, bound, f"expert {e}")
        at += c


@pytest.mark.parametrize("experts,average", [(64, 32), (40, 60), (16, 150), (48, 150)])
@pytest.mark.parametrize("swiglu", [False, True])
def test_experts_with_many_tiles_per_cta(cuda_device, experts, average, swiglu):
    """Several tiles per CTA, one after the other: from expert to expert, past
    empty experts and into the rows of none, 16 times bit by bit."""
    n, k, group = 2048, 768, 64
    g = torch.Generator(device="cpu")
    g.manual_seed(experts)
    counts = torch.randint(1, 2 * average, (experts,), generator=g)
    counts[torch.rand(experts, generator=g) < 0.2] = 0
    counts[0], counts[-1] = 0, average
    tail = 37
    ends = [0] + counts.cumsum(0).tolist()
    rows = ends[-1] + tail
    assert rows // experts > 8
    gd = torch.Generator(device=cuda_device)
    gd.manual_seed(experts)
    R = 2 * n if swiglu else n
    codes = torch.randint(-2 ** 31, 2 ** 31, (experts, R, k // 8), generator=gd, device=cuda_device).to(torch.int32)
    scales = ((torch.rand(experts, R, k // group, generator=gd, device=cuda_device) + 0.25) * 0.01).to(BF16)
    z = torch.randint(0, 16, (experts, R, k // group), generator=gd, device=cuda_device).to(torch.uint8)
    x = _x(rows, k, BF16, cuda_device, 3)
    offsets = torch.tensor(ends, dtype=torch.int32, device=cuda_device)
    call = quant.w4_expert_swiglu if swiglu else quant.w4_expert_linear
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    first = call(x, offsets, codes, scales, z, status=status)
    for _ in range(15):
        out = torch.full_like(first, float("nan"))
        assert torch.equal(call(x, offsets, codes, scales, z, out=out), first)
    assert int(status) == 0 and bool((first[rows - tail:] == 0).all())
    some = torch.arange(0, n, 13, device=cuda_device)
    pick = torch.cat([some, some + n]) if swiglu else some
    for e in range(experts):
        a, b = ends[e], ends[e + 1]
        w = quant.dequantize_w4(quant.W4Weight(codes[e, pick], scales[e, pick], z[e, pick]))
        ref, bound = product(x[a:b], w.to(BF16).double().cpu(), swiglu=swiglu, rows=1)
        check(first[a:b][:, some], ref, bound, f"expert {e}")
