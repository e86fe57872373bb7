"""CPU checks of the feed-forward operators: the 4-bit format, and the C ABI's
refusals (none of them reaches a launch)."""

import ctypes

import pytest
import torch

from aspire_b200 import _capi, moe, quant


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize_is_the_nearest_code(symmetric, group):
    g = torch.Generator()
    g.manual_seed(group)
    w = (torch.randn(3, 5, 256, generator=g) * 0.02).to(torch.bfloat16)
    w[0, 0] = 0
    w[1, 1] = 0.5
    q = quant.quantize_w4(w, group, symmetric)
    assert q.codes.shape == (3, 5, 32) and q.scales.shape == (3, 5, 256 // group) and q.group == group
    assert (q.zeros is None) == symmetric
    d = quant.dequantize_w4(q)
    step = q.scales.float().abs().repeat_interleave(group, -1)
    # Half a step to the nearest code; at the ends the stored scale's rounding
    # (2^-8) and the missing ninth positive code add up to a step.
    assert bool(((d - w.float()).abs() <= step * 1.1).all())
    assert bool((d[0, 0].abs() <= 1e-30).all())


def test_word_layout():
    codes = torch.zeros(1, 4, dtype=torch.int32)
    codes[0, 2] = 0x76543210
    scales = torch.ones(1, 1, dtype=torch.bfloat16)
    d = quant.dequantize_w4(quant.W4Weight(codes, scales, torch.zeros(1, 1, dtype=torch.uint8)))
    assert d[0, 16:24].tolist() == [0, 4, 1, 5, 2, 6, 3, 7]


def test_quantize_refusals():
    w = torch.zeros(4, 96, dtype=torch.bfloat16)
    for bad in (lambda: quant.quantize_w4(w, 64), lambda: quant.quantize_w4(w, 48), lambda: quant.quantize_w4(w.float(), 32),
                lambda: quant.quantize_w4(w[0], 32)):
        with pytest.raises(ValueError):
            bad()


def test_products_refuse_cpu_tensors():
    q = quant.quantize_w4(torch.ones(4, 64, dtype=torch.bfloat16), 32)
    with pytest.raises(ValueError):
        quant.w4_linear(torch.ones(1, 64, dtype=torch.bfloat16), q.codes, q.scales)


def _w4_args(**kw):
    a = _capi.AspireW4Args()
    fake = 1 << 20
    base = dict(x=fake, x_stride=256, rows=2, codes=fake, codes_stride=32, scales=fake, scales_stride=4, out=fake,
                out_stride=64, n=64, k=256, group=64, type=_capi.T_BF16)
    base.update(kw)
    for k, v in base.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [
    dict(type=0), dict(type=7), dict(n=0), dict(k=0), dict(rows=-1), dict(group=48), dict(group=0), dict(k=48, group=32),
    dict(group=96), dict(x=None), dict(codes=None), dict(scales=None), dict(out=None), dict(x=(1 << 20) + 2),
    dict(codes=(1 << 20) + 4), dict(x_stride=255), dict(x_stride=260), dict(codes_stride=33), dict(codes_stride=28),
    dict(scales_stride=3), dict(out_stride=63), dict(zeros=1 << 20, zeros_stride=1),
    dict(residual=1 << 20, residual_stride=3), dict(swiglu=1, residual=1 << 20, residual_stride=64),
    dict(offsets=1 << 20, experts=0), dict(offsets=1 << 20, experts=2, codes_stride_e=2)])
def test_w4_abi_refusals(built_library, bad):
    a = _w4_args(**bad)
    assert built_library.aspire_w4_linear(ctypes.byref(a), None) == _capi.ASPIRE_ERR_INVALID
    assert b"aspire_w4_linear" in built_library.aspire_last_error()


def test_w4_abi_no_rows(built_library):
    assert built_library.aspire_w4_linear(ctypes.byref(_w4_args(rows=0)), None) == _capi.ASPIRE_OK
    assert built_library.aspire_w4_linear(None, None) == _capi.ASPIRE_ERR_INVALID


def _set(a, base, bad):
    for k, v in {**base, **bad}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [
    dict(num_experts=0), dict(num_experts=513), dict(top_k=0), dict(top_k=33), dict(top_k=9), dict(tokens=-1),
    dict(tokens=1 << 31), dict(logits_type=3), dict(logits_stride=7), dict(offsets=None), dict(experts=None),
    dict(position=None), dict(source=None), dict(weights=None)])
def test_route_abi_refusals(built_library, bad):
    p = 1 << 20
    base = dict(logits=p, logits_stride=8, tokens=4, num_experts=8, top_k=2, weights=p, experts=p, position=p, source=p,
                offsets=p)
    a = _set(_capi.AspireMoeRouteArgs(), base, bad)
    assert built_library.aspire_moe_route(ctypes.byref(a), None) == _capi.ASPIRE_ERR_INVALID


def test_route_workspace(built_library):
    need = built_library.aspire_moe_route_workspace
    assert need(1024, 64, 8) == 0 and need(0, 64, 8) == 0
    assert need(1025, 64, 8) == 17 * 64 * 4  # blocks of 512 slots
    a = _set(_capi.AspireMoeRouteArgs(), dict(logits=1 << 20, logits_stride=64, tokens=1025, num_experts=64, top_k=8,
                                              weights=1 << 20, experts=1 << 20, position=1 << 20, source=1 << 20,
                                              offsets=1 << 20), {})
    assert built_library.aspire_moe_route(ctypes.byref(a), None) == _capi.ASPIRE_ERR_CAPACITY


@pytest.mark.parametrize("bad", [
    dict(type=5), dict(tokens=-1), dict(top_k=0), dict(top_k=33), dict(width=0), dict(width=4), dict(in_stride=60),
    dict(out_stride=68), dict(position=None), dict(offsets=None), dict(in_=None), dict(out=None), dict(in_=(1 << 20) + 8),
    dict(residual=1 << 20, residual_stride=8)])
def test_permute_abi_refusals(built_library, bad):
    p = 1 << 20
    base = dict(type=_capi.T_BF16, in_=p, in_stride=64, position=p, offsets=p, num_experts=4, top_k=2, tokens=3, width=64,
                out=p, out_stride=64)
    for name in ("aspire_moe_dispatch", "aspire_moe_combine"):
        a = _set(_capi.AspireMoePermuteArgs(), base, bad)
        assert getattr(built_library, name)(ctypes.byref(a), None) == _capi.ASPIRE_ERR_INVALID
    a = _set(_capi.AspireMoePermuteArgs(), base, {})
    assert built_library.aspire_moe_combine_grad(ctypes.byref(a), None) == _capi.ASPIRE_ERR_INVALID  # no gradient


def test_calls_refuse_what_is_not_a_tensor(built_library):
    with pytest.raises(ValueError, match="tensor"):
        quant.w4_linear([1.0], None, None)
    with pytest.raises(ValueError, match="tensor"):
        moe.moe_sort([[0, 1]], 2)
    with pytest.raises(ValueError, match="integer"):
        moe.moe_route(torch.zeros(2, 4), 1.5)
