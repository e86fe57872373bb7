"""GPU tests of where the feed-forward operators' operands and outputs lie:
outputs that overlap inputs, tensors' versions, row ranges that do not begin at
the first row, strides of broadcast and of size-one dimensions."""

import pytest
import torch

from aspire_b200 import moe, quant
from ffn_reference import check, product, random_w4

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _randn(*shape, dtype, device, seed):
    g = torch.Generator(device="cpu")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).to(device)


# ------------------------------------------------------------------ overlaps
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_products_refuse_outputs_that_overlap(cuda_device, rows):
    n = k = 64
    codes, scales, _, w = random_w4((n,), k, 32, False, BF16, cuda_device, seed=1)
    buf = _randn(rows + 1, 2 * k, dtype=BF16, device=cuda_device, seed=2)
    x = buf[:rows, :k]
    ref, bound = product(x, w)
    flat = buf.view(-1)
    shifted = flat[8:8 + rows * 2 * k].view(rows, 2 * k)[:, :n]
    outs = [shifted, flat[k - 1:k - 1 + n].view(1, n) if rows == 1 else buf[1:, :n]]
    for out in (x, *outs):
        with pytest.raises(ValueError, match="overlap"):
            quant.w4_linear(x, codes, scales, out=out)
    for out in outs:
        with pytest.raises(ValueError, match="overlap"):
            quant.w4_linear(x.clone(), codes, scales, residual=x, out=out)
    with pytest.raises(ValueError, match="overlap"):
        quant.w4_swiglu(x, codes, scales, out=x[:, n // 2:])
    # Interleaved with x and sharing nothing: allowed, at this pitch and at another.
    check(quant.w4_linear(x, codes, scales, out=buf[:rows, k:]), ref, bound)
    assert torch.equal(buf[:rows, k:], quant.w4_linear(x, codes, scales))
    # The residual itself: allowed.
    r = _randn(rows, n, dtype=BF16, device=cuda_device, seed=3)
    want = quant.w4_linear(x, codes, scales, residual=r)
    assert torch.equal(quant.w4_linear(x, codes, scales, residual=r, out=r), want)


@pytest.mark.parametrize("top_k", [1, 2])
def test_combine_refuses_outputs_that_overlap(cuda_device, top_k):
    tokens, width = 6, 64
    chosen = torch.arange(tokens * top_k, device=cuda_device, dtype=torch.int32).view(tokens, top_k) % 4
    order = moe.moe_sort(chosen, 4)
    buf = _randn(tokens * top_k + 1, 2 * width, dtype=torch.float32, device=cuda_device, seed=4)
    rows, weights = buf[:tokens * top_k, :width], torch.full((tokens, top_k), 0.5, device=cuda_device)
    res = _randn(tokens + 1, width, dtype=torch.float32, device=cuda_device, seed=5)
    for kw in (dict(out=rows[:tokens]), dict(out=buf[1:1 + tokens, :width]),
               dict(out=buf[:tokens, 4:4 + width]), dict(residual=res[:tokens], out=res[1:])):
        with pytest.raises(ValueError, match="overlap"):
            moe.moe_combine(rows, weights, order, **kw)
    want = moe.moe_combine(rows, weights, order, residual=res[:tokens])
    assert torch.equal(moe.moe_combine(rows, weights, order, residual=res[:tokens], out=buf[:tokens, width:]), want)
    assert torch.equal(moe.moe_combine(rows, weights, order, residual=res[:tokens], out=res[:tokens]), want)


def test_written_outputs_change_their_version(cuda_device):
    codes, scales, _, _ = random_w4((64,), 64, 32, False, BF16, cuda_device, seed=1)
    x = _randn(3, 64, dtype=BF16, device=cuda_device, seed=2)
    order = moe.moe_sort(torch.zeros(3, 1, dtype=torch.int32, device=cuda_device), 2)
    weights = torch.ones(3, 1, device=cuda_device)
    for write in (lambda out: quant.w4_linear(x, codes, scales, out=out),
                  lambda out: quant.w4_swiglu(x, codes.repeat(2, 1), scales.repeat(2, 1), out=out),
                  lambda out: moe.moe_combine(x, weights, order, out=out)):
        leaf = _randn(3, 64, dtype=BF16, device=cuda_device, seed=3).requires_grad_()
        out = torch.zeros(3, 64, dtype=BF16, device=cuda_device)
        saved = leaf * out  # keeps `out` for the backward pass
        before = out._version
        write(out)
        assert out._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            saved.sum().backward()
        with pytest.raises(ValueError, match="out requires"):
            write(leaf)
        with torch.no_grad():
            write(leaf)


# ---------------------------------------------------------------- row ranges
@pytest.mark.parametrize("head,counts,tail", [
    (1, [2, 0, 3], 0), (9, [1, 7, 0], 4), (40, [3], 0), (12, [0, 0], 0),                    # few rows per expert
    (3, [60, 0, 20], 0), (200, [30, 1], 5), (131, [0, 140], 70), (290, [0], 0)])            # many
@pytest.mark.parametrize("n,k,group,zeros,dtype,swiglu", [
    (72, 288, 32, True, BF16, False), (296, 640, 128, False, BF16, True), (130, 2048, 64, True, F16, False)])
def test_rows_before_the_first_expert_give_zero(cuda_device, head, counts, tail, n, k, group, zeros, dtype, swiglu):
    """Offsets of a share of the experts, as a rank that holds only those has
    them: the rows before belong to none of them, like the rows past the last."""
    E, rows = len(counts), head + sum(counts) + tail
    codes, scales, z, w = random_w4((E, 2 * n if swiglu else n), k, group, zeros, dtype, cuda_device, seed=E + n)
    x = _randn(rows, k, dtype=dtype, device=cuda_device, seed=5)
    offsets = (torch.tensor([0] + counts).cumsum(0) + head).to(torch.int32).to(cuda_device)
    call = quant.w4_expert_swiglu if swiglu else quant.w4_expert_linear
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    y = call(x, offsets, codes, scales, z, out=torch.full((rows, n), float("nan"), dtype=dtype, device=cuda_device),
             status=status)
    assert bool((y[:head] == 0).all()) and bool((y[rows - tail:] == 0).all())
    at = head
    for e, c in enumerate(counts):
        ref, bound = product(x[at:at + c], w[e], swiglu=swiglu, rows=rows if -(-rows // E) > 8 else 1)
        check(y[at:at + c], ref, bound, f"expert {e}")
        at += c
    assert int(status) == 0


# ------------------------------------------------------------------- strides
@pytest.mark.parametrize("rows", [6, 100])
@pytest.mark.parametrize("swiglu", [False, True])
def test_one_matrix_for_all_experts(cuda_device, rows, swiglu):
    """An expert stride of 0, whatever the row count."""
    E, n, k = 3, 96, 512
    codes, scales, z, _ = random_w4((2 * n if swiglu else n,), k, 64, True, BF16, cuda_device, seed=1)
    many = [t[None].expand(E, *t.shape) for t in (codes, scales, z)]
    assert many[0].stride(0) == 0
    x = _randn(rows, k, dtype=BF16, device=cuda_device, seed=2)
    offsets = torch.tensor([0, rows // 3, rows // 2, rows], dtype=torch.int32, device=cuda_device)
    call = quant.w4_expert_swiglu if swiglu else quant.w4_expert_linear
    assert torch.equal(call(x, offsets, *many), call(x, offsets, *(t.contiguous() for t in many)))


@pytest.mark.parametrize("rows", [2, 40])
def test_strides_of_size_one_dimensions_do_not_matter(cuda_device, rows):
    k, group = 256, 64
    codes, scales, z, _ = random_w4((1,), k, group, True, BF16, cuda_device, seed=3)
    x = _randn(rows, k, dtype=BF16, device=cuda_device, seed=4)
    want = quant.w4_linear(x, codes, scales, z)
    odd = [t.as_strided(t.shape, (3, 1)) for t in (codes, scales, z)]
    assert torch.equal(quant.w4_linear(x, *odd), want)
    offsets = torch.tensor([0, rows], dtype=torch.int32, device=cuda_device)
    one = [t.as_strided((1, *t.shape), (1, 3, 1)) for t in (codes, scales, z)]
    assert torch.equal(quant.w4_expert_linear(x, offsets, *one),
                       quant.w4_expert_linear(x, offsets, codes[None], scales[None], z[None]))
