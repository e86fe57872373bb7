"""CPU checks of a tree-speculation step's operators: refused arguments, at the
Python calls and at the C ABI.  Nothing is launched."""

import ctypes

import pytest
import torch

from aspire_b200 import _capi
from aspire_b200.kv_ops import build_step_tables, qkv_prologue
from aspire_b200.logits import adjust_logits, pick_tokens
from aspire_b200.tree import accept_tree

P = ctypes.c_void_p(256).value  # an address that no refused call reads


def _refused(lib, rc, text):
    assert rc == _capi.ASPIRE_ERR_INVALID
    assert text in lib.aspire_last_error().decode()


def test_python_calls_need_cuda_tensors(built_library):
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="CUDA"):
        build_step_tables(i32(1), None, i32(1, 2)[None], i32(0), i32(3), i32(1), tokens=0)
    with pytest.raises(ValueError, match="max_nodes"):
        build_step_tables(i32(1), None, i32(1, 2)[None], i32(0), i32(3), i32(1), tokens=1, parents=i32(-1))
    for call in (adjust_logits, pick_tokens):
        with pytest.raises(ValueError, match="CUDA"):
            call(torch.zeros(1, 4))
    with pytest.raises(ValueError, match="CUDA"):
        accept_tree(i32(1), i32(-1), i32(2), i32(0, 1), i32(0), 4)


def test_step_tables_abi(built_library):
    lib = built_library
    _refused(lib, lib.aspire_step_tables(None, None), "null")

    def args(**kw):
        a = _capi.AspireStepTablesArgs()
        a.rows, a.page_size, a.block_table_cols, a.tokens, a.free_capacity = 1, 16, 4, 2, 4
        for f in ("lengths", "block_table", "held", "free_pages", "free_count", "qo_indptr", "kv_indptr", "kv_len",
                  "last_page_len", "positions", "slots"):
            setattr(a, f, P)
        for k, v in kw.items():
            setattr(a, k, v)
        return ctypes.byref(a)

    for kw, text in [(dict(rows=-1), "range"), (dict(tokens=-1), "range"), (dict(page_size=0), "page_size"),
                     (dict(free_capacity=-1), "range"), (dict(block_table_cols=-1), "range"), (dict(block_table_cols=2 ** 22), "range"), (dict(lengths=None), "null"),
                     (dict(block_table=None), "null"), (dict(held=None), "null"), (dict(free_count=None), "null"),
                     (dict(free_pages=None), "null"), (dict(kv_len=None), "null"), (dict(positions=None), "positions"),
                     (dict(slots=None), "slots"), (dict(parents=P), "mask"), (dict(tree_mask_words=1), "parents"),
                     (dict(parents=P, tree_mask_words=2), "mask")]:
        _refused(lib, lib.aspire_step_tables(args(**kw), None), text)


def test_adjust_logits_abi(built_library):
    lib = built_library
    _refused(lib, lib.aspire_adjust_logits(None, None), "null")

    def args(**kw):
        a = _capi.AspireLogitsArgs()
        a.logits, a.logits_stride, a.type, a.tokens, a.vocab, a.rows, a.out, a.out_stride = P, 100, 1, 2, 100, 2, P, 100
        for k, v in kw.items():
            setattr(a, k, v)
        return ctypes.byref(a)

    for kw, text in [(dict(type=3), "type"), (dict(type=-1), "type"), (dict(vocab=0), "vocab"), (dict(rows=65535), "rows"),
                     (dict(tokens=-1), "range"), (dict(out=None), "either"), (dict(ids=P), "either"),
                     (dict(vocab=2 ** 30 + 1, logits_stride=2 ** 31, out_stride=2 ** 31), "2^30"), (dict(logits=None), "null"),
                     (dict(logits_stride=99), "apart"), (dict(out_stride=99), "apart"), (dict(rows=1), "indptr"),
                     (dict(history=P), "history_len"), (dict(tree_mask=P), "step_tokens"),
                     (dict(tree_mask=P, step_tokens=P), "words"), (dict(bias_indptr=P, bias_entries=3), "bias"),
                     (dict(bias_indptr=P, bias_entries=-1), "bias"), (dict(allowed=P, allowed_stride=3), "allowed")]:
        _refused(lib, lib.aspire_adjust_logits(args(**kw), None), text)
    assert lib.aspire_adjust_logits(args(tokens=0, rows=0), None) == _capi.ASPIRE_OK


def test_tree_accept_abi(built_library):
    lib = built_library
    _refused(lib, lib.aspire_tree_accept(None, None), "null")
    caches = (ctypes.c_void_p * 1)(P)
    odd = (ctypes.c_void_p * 1)(P + 8)

    def args(**kw):
        a = _capi.AspireTreeAcceptArgs()
        for f in ("tokens", "parents", "targets", "indptr", "lengths", "count", "path", "out_tokens"):
            setattr(a, f, P)
        a.new_lengths = P + 64
        a.total, a.rows, a.max_path = 3, 1, 4
        a.caches, a.num_caches, a.pages, a.page_size, a.token_bytes = caches, 1, 2, 16, 256
        a.block_table, a.block_table_cols = P, 2
        for k, v in kw.items():
            setattr(a, k, v)
        return ctypes.byref(a)

    for kw, text in [(dict(rows=-1), "range"), (dict(total=-1), "range"), (dict(max_path=0), "max_path"),
                     (dict(max_path=65), "max_path"), (dict(num_caches=129), "128"), (dict(num_caches=-1), "128"),
                     (dict(tokens=None), "null"), (dict(path=None), "null"), (dict(new_lengths=P), "new_lengths"),
                     (dict(block_table=None), "block table"), (dict(page_size=0), "geometry"),
                     (dict(token_bytes=24), "multiple of 16"), (dict(token_bytes=0), "multiple of 16"),
                     (dict(caches=odd), "aligned")]:
        _refused(lib, lib.aspire_tree_accept(args(**kw), None), text)
    assert lib.aspire_tree_accept(args(rows=0), None) == _capi.ASPIRE_OK


def test_tree_attention_abi(built_library):
    lib = built_library
    info = _capi.AspirePlanInfo()
    info.tc_enabled, info.max_q_len, info.num_qo_heads, info.num_kv_heads = 1, 40, 8, 2

    def call(mask=P, words=2, plan=None, **kw):
        a = _capi.AspireAttnArgs()
        a.num_qo_heads, a.num_kv_heads, a.head_dim, a.page_size = 8, 2, 128, 16
        for k, v in kw.items():
            setattr(a, k, v)
        for k, v in (plan or {}).items():
            setattr(info, k, v)
        return lib.aspire_tree_attention(ctypes.byref(a), mask, words, ctypes.byref(info), None)

    _refused(lib, call(mask=None), "null")
    _refused(lib, call(words=0), "mask_words")
    _refused(lib, call(words=1), "more queries")
    _refused(lib, call(dump=P), "dump")
    _refused(lib, call(num_qo_heads=98), "48")
    _refused(lib, call(), "null tensor")
    _refused(lib, call(plan=dict(tc_enabled=0)), "routing")
    _refused(lib, call(plan=dict(tc_enabled=1, causal=1)), "causal")


@pytest.mark.parametrize("group", [1, 3, 4, 8, 17, 48])
@pytest.mark.parametrize("rows", [[(100, 5)], [(5000, 12), (0, 3), (77, 0), (900, 40)], [(40000, 16)] * 3,
                                  [(3000, 100), (128, 64), (64, 1)] * 4])
def test_plans_for_trees_cover_every_key_once(built_library, rows, group):
    import numpy as np

    i32 = lambda a: np.ascontiguousarray(a, dtype=np.int32)  # noqa: E731
    ptr = lambda a: a.ctypes.data_as(_capi.c_int32_p)  # noqa: E731
    qo = i32(np.cumsum([0] + [n for _, n in rows]))
    kvl = i32([a + n for a, n in rows])
    kvp = i32(np.cumsum([0] + [-(-k // 16) for k in kvl]))
    buf = np.zeros(1 << 23, dtype=np.uint8)
    info = _capi.AspirePlanInfo()
    rc = built_library.aspire_plan_host_only(ptr(qo), ptr(kvp), ptr(kvl), len(kvl), 2 * group, 2, 128, 16,
                                             _capi.PLAN_TREE, 148, buf.ctypes.data_as(ctypes.c_void_p), buf.nbytes,
                                             1 << 31, ctypes.byref(info))
    assert rc == 0 and info.causal == _capi.PLAN_TREE
    w = buf.view(np.int32)
    assert w[10] == 0  # not causal
    items = w[w[5]:w[5] + 16 * info.num_items].reshape(-1, 16)
    seen = {}
    for row, head, _, q_len, _, kv_len, t0, t1, p0, p1, chunk, chunks, base, merge, kind, cols in items.tolist():
        assert kind == (2 if q_len * group > 64 else 1)
        assert 0 < p1 - p0 <= (256 if kind == 2 else 64) and p0 % group == 0
        assert t0 % 128 == 0 and cols <= 64 and (merge >= 0) == (chunks > 1)
        seen.setdefault((row, head, p0, p1), []).append((t0, t1))
    for b, (a, n) in enumerate(rows):
        for h in range(2):
            tiles = sorted(k for k in seen if k[:2] == (b, h))
            assert [t[2] for t in tiles] + [n * group] == [0] + [t[3] for t in tiles] or n == 0
            for t in tiles:
                ranges = sorted(seen[t])
                assert ranges[0][0] == 0 and ranges[-1][1] == a + n
                assert all(x[1] == y[0] for x, y in zip(ranges, ranges[1:]))


@pytest.mark.parametrize("room", [0, 100_000, 1_000_000, 1 << 31])
@pytest.mark.parametrize("rows", [[(5000, 12), (900, 40)], [(130000, 4)], [(600, 80)] * 48])
def test_plans_for_trees_fit_the_float_workspace(built_library, rows, room):
    import numpy as np

    i32 = lambda a: np.ascontiguousarray(a, dtype=np.int32)  # noqa: E731
    ptr = lambda a: a.ctypes.data_as(_capi.c_int32_p)  # noqa: E731
    qo = i32(np.cumsum([0] + [n for _, n in rows]))
    kvl = i32([a + n for a, n in rows])
    kvp = i32(np.cumsum([0] + [-(-k // 16) for k in kvl]))
    buf = np.zeros(1 << 23, dtype=np.uint8)
    info = _capi.AspirePlanInfo()
    rc = built_library.aspire_plan_host_only(ptr(qo), ptr(kvp), ptr(kvl), len(kvl), 64, 8, 128, 16, _capi.PLAN_TREE,
                                             148, buf.ctypes.data_as(ctypes.c_void_p), buf.nbytes, room,
                                             ctypes.byref(info))
    assert rc == 0 and info.float_bytes <= room


def test_prologue_at_abi(built_library):
    lib = built_library
    a = _capi.AspirePrologueArgs()
    _refused(lib, lib.aspire_qkv_prologue_at(ctypes.byref(a), None, None), "positions")


def test_the_prologue_of_trees_refuses_gradients_and_overlaps():
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    q, k, v = (torch.zeros(4, h, 128, dtype=torch.bfloat16) for h in (2, 1, 1))
    cache = torch.zeros(2, 2, 16, 1, 128, dtype=torch.bfloat16)
    w = torch.ones(128, dtype=torch.bfloat16)
    rows = (i32(0, 4), None), (cache, i32(0), i32(0, 1), i32(4))

    def call(q=q, k=k, v=v, cache=cache, w=w, positions=i32(0, 1, 1, 2), **kw):
        return qkv_prologue(q, k, v, *rows[0], cache, *rows[1][1:], q_norm_weight=w, k_norm_weight=w, positions=positions, **kw)

    for name, t in (("q", q), ("k", k), ("v", v), ("cache", cache), ("w", w), ("q_out", q)):
        with pytest.raises(ValueError, match="gradient"):
            call(**{name: t.clone().requires_grad_()})
    for name, t in (("q_out", torch.zeros_like(q)), ("cache", torch.zeros_like(cache))):
        with pytest.raises(ValueError, match="overlap"):
            call(positions=t.view(-1).view(torch.int32)[100:104], **{name: t})
