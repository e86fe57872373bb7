"""The feed-forward operators refuse what would lose a derivative (checked
before anything reaches a device)."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

from aspire_b200 import moe, quant

BF16 = torch.bfloat16


def _product_operands():
    w = quant.quantize_w4(torch.ones(8, 64, dtype=BF16), 32)
    return torch.ones(2, 64, dtype=BF16), w


@pytest.mark.parametrize("who", ["x", "scales", "residual"])
def test_products_refuse_operands_that_require_a_gradient(built_library, who):
    x, w = _product_operands()
    residual = torch.ones(2, 8, dtype=BF16)
    dict(x=x, scales=w.scales, residual=residual)[who].requires_grad_()
    with pytest.raises(ValueError, match="no gradient"):
        quant.w4_linear(x, w.codes, w.scales, residual=residual)
    if who == "x":
        offsets = torch.tensor([0, 2], dtype=torch.int32)
        with pytest.raises(ValueError, match="no gradient"):
            quant.w4_swiglu(x, w.codes, w.scales)
        for call in (quant.w4_expert_linear, quant.w4_expert_swiglu):
            with pytest.raises(ValueError, match="no gradient"):
                call(x, offsets, w.codes[None], w.scales[None])
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        quant.w4_linear(x, w.codes, w.scales, residual=residual)


def test_a_layer_with_a_gradient_through_its_experts_is_refused(built_library):
    x, w = _product_operands()
    rows = (x.requires_grad_() * 1)  # what a dispatch with a gradient returns
    with pytest.raises(ValueError, match="no gradient"):
        quant.w4_expert_swiglu(rows, torch.tensor([0, 2], dtype=torch.int32), w.codes[None], w.scales[None])


def test_tangents_are_refused(built_library):
    x, w = _product_operands()
    order = moe.ExpertOrder(torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32),
                            torch.zeros(2, dtype=torch.int32))
    weights = torch.ones(2, 1)
    with fwad.dual_level():
        dual = fwad.make_dual(x, torch.ones_like(x))
        dual_weights = fwad.make_dual(weights, torch.ones_like(weights))
        for call in (lambda: quant.w4_linear(dual, w.codes, w.scales), lambda: moe.moe_route(dual, 2),
                     lambda: moe.moe_dispatch(dual, order), lambda: moe.moe_combine(dual, weights, order),
                     lambda: moe.moe_combine(x, dual_weights, order),
                     lambda: moe.moe_combine(x, weights, order, residual=dual)):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
