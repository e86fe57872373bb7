"""CPU checks of the size limits of the 4-bit products (none reaches a launch)."""

import ctypes

import pytest

from aspire_b200 import _capi


def _args(**kw):
    a = _capi.AspireW4Args()
    fake = 1 << 20
    base = dict(x=fake, x_stride=kw["k"], rows=2, codes=fake, codes_stride=kw["k"] // 8, scales=fake,
                scales_stride=kw["k"] // kw["group"], out=fake << 4, out_stride=64, n=64, type=_capi.T_BF16)
    base.update(kw)
    for k, v in base.items():
        setattr(a, k, v)
    return a


def _group_of(block, blocks_per_group):
    """The kernels' quotient: a multiplication by floor(2^32 / m) + 1."""
    return (block * ((1 << 32) // blocks_per_group + 1)) >> 32


@pytest.mark.parametrize("k,group,block", [
    (1 << 29, 1 << 28, 4192257), (1 << 29, 1 << 23, 3997636), (3 << 24, 1 << 24, 262137)])
def test_groups_that_the_kernels_would_confuse_are_refused(built_library, k, group, block):
    assert block < k // 128 and _group_of(block, group // 128) != block // (group // 128)
    assert built_library.aspire_w4_linear(ctypes.byref(_args(k=k, group=group)), None) == _capi.ASPIRE_ERR_INVALID
    assert b"2^46" in built_library.aspire_last_error()


@pytest.mark.parametrize("m", [2, 3, 7, 1000, 1025, 4095, 4097, 65535])
def test_accepted_groups_are_exact(m):
    blocks = min((1 << 32) // m, 1 << 22)
    for block in (*range(min(blocks, 20000)), *range(max(0, blocks - 20000), blocks)):
        assert _group_of(block, m) == block // m


def test_rows_past_the_counts_are_refused(built_library):
    for kw in (dict(rows=(1 << 31) - 1), dict(rows=(1 << 31) - 128),
               dict(rows=1 << 30, offsets=1 << 20, experts=1024, codes_stride_e=2048)):
        assert built_library.aspire_w4_linear(ctypes.byref(_args(k=32, group=32, **kw)), None) == _capi.ASPIRE_ERR_INVALID
