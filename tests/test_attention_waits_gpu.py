"""Bounded waits of the tcgen05 attention kernel that expire at different places:
every launch ends, reports a timeout or is right, and leaves nothing behind."""

import pytest
import torch

from aspire_b200 import _capi
from aspire_b200.attention import HolisticAttentionWrapper
from aspire_b200.workloads import fill_tensors, make_layout, rows_layout
from gpu_helpers import assert_attention_close, oracle_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["decode", "prefill", "both"])
def test_waits_that_expire_at_different_places(cuda_device, built_library, kind):
    dev = cuda_device
    if kind == "decode":
        lay = make_layout(batch=16, ctx=4096, num_qo_heads=32, num_kv_heads=8, draft_fraction=0.5, budget_pages=64,
                          seed=81)
    elif kind == "prefill":
        lay = rows_layout([300, 200], [2048, 1024], 32, 8, seed=82)
    else:
        lay = rows_layout([256, 1, 5, 1], [1024, 2048, 3000, 700], 32, 8, seed=83)
    q, kv = fill_tensors(lay, device=dev, seed=84)
    w = HolisticAttentionWrapper(torch.empty(1, device=dev))
    ref_out, ref_lse, _ = oracle_attention(lay, q, kv)

    def run():
        w.plan_host(torch.from_numpy(lay.qo_indptr), torch.from_numpy(lay.kv_indptr), torch.from_numpy(lay.kv_lens),
                    torch.from_numpy(lay.kv_indices).to(dev), lay.num_qo_heads, lay.num_kv_heads, 128, 16, causal=True)
        w.clear_device_status()
        out, lse = w.run(q, kv, return_lse=True)
        torch.cuda.synchronize()
        return out, lse, w.device_status()

    expired = 0
    for limit in (1, 500, 2000, 4000, 8000, 16000):
        for _ in range(5):
            _capi.check(built_library.aspire_set_wait_limit_ns(limit), "aspire_set_wait_limit_ns")
            try:
                out, lse, status = run()
            finally:
                _capi.check(built_library.aspire_set_wait_limit_ns(0), "aspire_set_wait_limit_ns")
            assert status in (0, _capi.STATUS_TIMEOUT)
            expired += status != 0
            if status == 0:
                assert_attention_close(out, lse, ref_out, ref_lse)
            out, lse, status = run()
            assert status == 0
            assert_attention_close(out, lse, ref_out, ref_lse)
    assert expired


def test_expired_waits_leave_no_copy_behind(cuda_device, built_library):
    """Short items, whose producers issue all their copies without a wait, stopped
    by expired waits and followed at once by a launch on the same shared memory."""
    dev = cuda_device
    short = rows_layout([1, 3, 5] * 20, [200, 130, 250] * 20, 32, 8, seed=85)
    other = make_layout(batch=16, ctx=4096, num_qo_heads=32, num_kv_heads=8, draft_fraction=0.5, budget_pages=64, seed=86)
    run = []
    for lay in (short, other):
        q, kv = fill_tensors(lay, device=dev, seed=87)
        w = HolisticAttentionWrapper(torch.empty(1, device=dev))
        w.plan_host(torch.from_numpy(lay.qo_indptr), torch.from_numpy(lay.kv_indptr), torch.from_numpy(lay.kv_lens),
                    torch.from_numpy(lay.kv_indices).to(dev), lay.num_qo_heads, lay.num_kv_heads, 128, 16, causal=True)
        run.append((w, q, kv, lay))
    (w, q, kv, _), (w2, q2, kv2, lay2) = run
    ref_out, ref_lse, _ = oracle_attention(lay2, q2, kv2)
    for _ in range(10):
        _capi.check(built_library.aspire_set_wait_limit_ns(1), "aspire_set_wait_limit_ns")
        try:
            w.run(q, kv)
        finally:
            _capi.check(built_library.aspire_set_wait_limit_ns(0), "aspire_set_wait_limit_ns")
        w2.clear_device_status()
        w2.plan_host(torch.from_numpy(lay2.qo_indptr), torch.from_numpy(lay2.kv_indptr), torch.from_numpy(lay2.kv_lens),
                     torch.from_numpy(lay2.kv_indices).to(dev), lay2.num_qo_heads, lay2.num_kv_heads, 128, 16, causal=True)
        out, lse = w2.run(q2, kv2, return_lse=True)
        torch.cuda.synchronize()
        assert w2.device_status() == 0
        assert_attention_close(out, lse, ref_out, ref_lse)
