"""GPU tests of the tcgen05 products' bounded waits and of the hand-over of
their stages."""

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


@pytest.fixture
def short_waits(built_library):
    """Sets the limit of a wait in nanoseconds; the default comes back at the end."""
    yield built_library.aspire_set_wait_limit_ns
    built_library.aspire_set_wait_limit_ns(0)


@pytest.mark.parametrize("limit", [1, 2000, 5000, 10000])
@pytest.mark.parametrize("experts", [0, 16])
def test_expired_waits_with_many_tiles_per_cta(cuda_device, short_waits, experts, limit):
    """Each CTA has several tiles, so that the wait for the previous tile's sums
    is among those that can expire, at different places by the limit.  Every
    call ends; one that reports no timeout is right, and so is the next call
    with the default limit."""
    n, k, rows = 3000 if experts else 9000, 512, 2400
    codes, scales, z, _ = random_w4((experts, n) if experts else (n,), k, 64, True, BF16, cuda_device, seed=limit)
    x = _x(rows, k, BF16, cuda_device, 3)
    offsets = (torch.arange(experts + 1) * (rows // max(experts, 1))).to(torch.int32).to(cuda_device)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)

    def call():
        if experts:
            return quant.w4_expert_linear(x, offsets, codes, scales, z, status=status)
        return quant.w4_linear(x, codes, scales, z, status=status)
    want = call()
    assert int(status) == 0
    for _ in range(4):
        status.zero_()
        short_waits(limit)
        got = call()
        torch.cuda.synchronize()
        short_waits(0)
        assert int(status) == 8 or (int(status) == 0 and torch.equal(got, want))
        status.zero_()
        assert torch.equal(call(), want) and int(status) == 0


@pytest.mark.parametrize("rows,n,k", [(40, 512, 4096), (300, 256, 1024), (64, 1024, 512)])
def test_expired_waits_leave_no_copy_behind(cuda_device, short_waits, rows, n, k):
    """The producers of these calls (few stages per CTA, clusters) issue all their
    copies without a wait, and another role stops the CTA after that.  The next
    launches take the same shared memory at once: a copy that landed late would
    change their results."""
    codes, scales, z, _ = random_w4((n,), k, 64, True, BF16, cuda_device, seed=4)
    x = _x(rows, k, BF16, cuda_device, 5)
    other_codes, other_scales, other_z, _ = random_w4((1024,), 2048, 64, True, BF16, cuda_device, seed=6)
    other_x = _x(96, 2048, BF16, cuda_device, 7)
    want = quant.w4_linear(other_x, other_codes, other_scales, other_z)
    mine = quant.w4_linear(x, codes, scales, z)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    for _ in range(25):
        status.zero_()
        short_waits(1)
        got = quant.w4_linear(x, codes, scales, z, status=status)
        short_waits(0)
        after = [quant.w4_linear(other_x, other_codes, other_scales, other_z) for _ in range(2)]
        assert int(status) == 8 or torch.equal(got, mine)
        assert all(torch.equal(a, want) for a in after)
    assert torch.equal(quant.w4_linear(x, codes, scales, z), mine)


@pytest.mark.parametrize("rows", [32, 64, 300])
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_every_variant_repeats_bit_by_bit(cuda_device, rows, swiglu, group, dtype):
    """All 36 forms of the kernel with two tiles and more per CTA: a stage that is
    released before its codes have been read shows in some of the runs."""
    R, k = 80000, 1024
    g = torch.Generator(device=cuda_device)
    g.manual_seed(group + rows)
    codes = torch.randint(-2 ** 31, 2 ** 31, (R, k // 8), generator=g, device=cuda_device).to(torch.int32)
    scales = ((torch.rand(R, k // group, generator=g, device=cuda_device) + 0.25) * 0.01).to(dtype)
    z = torch.randint(0, 16, (R, k // group), generator=g, device=cuda_device).to(torch.uint8)
    x = _x(rows, k, dtype, cuda_device, 3)
    call = quant.w4_swiglu if swiglu else quant.w4_linear
    first = call(x, codes, scales, z)
    for _ in range(15):
        assert torch.equal(call(x, codes, scales, z), first)
    n = first.shape[1]
    some = torch.arange(0, n, n // 300 + 1, device=cuda_device)  # features of every tile
    pick = torch.cat([some, some + n]) if swiglu else some
    w = quant.dequantize_w4(quant.W4Weight(codes[pick], scales[pick], z[pick])).double().cpu()
    ref, bound = product(x, w, swiglu=swiglu)
    check(first[:, some], ref, bound)
