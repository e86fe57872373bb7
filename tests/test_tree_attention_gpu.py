"""Attention of trees of drafted tokens over the paged cache (``run`` with a
tree mask) against the definition in 64 bits, with the bound of the kernels'
roundings."""

import math
import random

import pytest
import torch

from aspire_b200 import _capi
from aspire_b200.attention import HolisticAttentionWrapper, first_last_dump_jit_args
import tree_reference as ref

pytestmark = pytest.mark.gpu


class Case:
    """Rows of (keys before the nodes, nodes); masks by `kind`: trees, random
    bits, nothing, everything."""

    def __init__(self, dev, rows, heads, kv_heads, kind="tree", seed=0, extra_words=0, pad=0, scale=1.0, pages_pad=3):
        rng = random.Random(seed)
        g = torch.Generator().manual_seed(seed)
        nodes = [n for _, n in rows]
        self.ends = [a + n for a, n in rows]
        self.starts = ref.indptr(nodes)
        total = self.starts[-1] + pad
        per = [-(-e // 16) for e in self.ends]
        order = list(range(sum(per) + pages_pad))
        rng.shuffle(order)
        at = ref.indptr(per)
        self.kv_indptr = at
        self.pages = [order[at[b]:at[b + 1]] for b in range(len(rows))]
        self.cache = torch.randn(len(order), 2, 16, kv_heads, 128, generator=g).to(torch.bfloat16)
        # Places behind a row's end hold what an earlier owner of the page left.
        for b, e in enumerate(self.ends):
            if e % 16:
                self.cache[self.pages[b][-1], :, e % 16:] = math.nan
        self.q = (torch.randn(total, heads, 128, generator=g) * scale).to(torch.bfloat16)
        words = (max(nodes + [1]) + 31) // 32 + extra_words
        self.seen, mask = [], []
        for n in nodes:
            s = torch.zeros(n, n, dtype=torch.bool)
            if kind == "tree" and n:
                for i, path in enumerate(ref.ancestors(ref.random_parents(rng, n))):
                    s[i, path] = True
            elif kind == "random":
                s = torch.rand(n, n, generator=g) < 0.4
            elif kind == "all":
                s[:] = True
            elif kind == "chain":
                s = torch.ones(n, n).tril().bool()
            self.seen.append(s)
            mask += ref.mask_words([r.nonzero()[:, 0].tolist() for r in s], words)
        mask += [[-1] * words] * pad
        self.mask = torch.tensor(mask, dtype=torch.int32, device=dev).view(total, words)
        self.dev, self.heads, self.kv_heads, self.rows = dev, heads, kv_heads, rows

    def plan(self, device_plan=False, tables=False, wrapper=None, trees=False):
        i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
        w = wrapper or HolisticAttentionWrapper(torch.empty(1, device=self.dev))
        flat = i32([p for r in self.pages for p in r] or [0]).to(self.dev)
        if tables:
            cols = max(len(r) for r in self.pages)
            t = i32([r + [10 ** 6] * (cols - len(r)) for r in self.pages]).to(self.dev)
            w.set_page_tables(torch.ones(len(self.rows), dtype=torch.int32, device=self.dev), t, t)
            flat = None
        shape = (self.heads, self.kv_heads, 128, 16)
        if device_plan:
            last = i32([(e - 1) % 16 + 1 if e else 0 for e in self.ends]).to(self.dev)
            w.plan_device(i32(self.starts).to(self.dev), i32(self.kv_indptr).to(self.dev), last, *shape,
                          paged_kv_indices=flat, causal=False, trees=trees)
        else:
            w.plan_host(i32(self.starts), i32(self.kv_indptr), i32(self.ends), flat, *shape, causal=False, trees=trees)
        return w

    def check(self, out, lse, rows=None):
        exp, else_, bound, lbound = ref.tree_attention(self.q, self.cache.nan_to_num(0), self.pages, self.starts,
                                                       self.ends, self.seen)
        n = self.starts[-1]
        d = (out.double().cpu() - exp).abs()[:n]
        bad = ~(d <= bound[:n])
        assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} out, worst {(d / bound[:n].clamp(min=1e-300)).max():.3g}"
        none = else_[:n] == -math.inf
        got = lse.double().cpu()[:n]
        assert torch.equal(got == -math.inf, none)
        assert bool((out.cpu()[:n][none] == 0).all())
        assert bool(((got - else_[:n]).abs()[~none] <= lbound[:n][~none]).all())

    def run(self, **kw):
        w = self.plan(**kw)
        out, lse = w.run(self.q.to(self.dev), self.cache.to(self.dev), tree_mask=self.mask, return_lse=True)
        assert w.device_status() == 0
        return out, lse


ROWS = {
    "one": [(0, 1)],
    "short": [(130, 5)],
    "no_prefix": [(0, 7), (0, 33), (0, 1)],
    "tile_edges": [(128 - 3, 6), (128, 9), (127, 2), (64 - 5, 12), (256 - 16, 16), (1, 127)],
    "idle_rows": [(40, 0), (300, 11), (0, 0), (17, 3)],
    "ragged": [(700, 13), (33, 31), (1000, 20), (5, 8), (511, 1)],
    "split": [(3001, 9)],
    "wide": [(900, 64), (100, 33), (1, 100), (63, 65)],
    "more_than_an_item": [(200, 140)],
}


@pytest.mark.parametrize("heads,kv_heads", [(4, 1), (8, 8), (10, 2)])
@pytest.mark.parametrize("rows", list(ROWS))
def test_trees(cuda_device, rows, heads, kv_heads):
    c = Case(cuda_device, ROWS[rows], heads, kv_heads, seed=len(rows) * 7 + heads)
    c.check(*c.run())


@pytest.mark.parametrize("heads,kv_heads", [(16, 2), (48, 1), (17, 1), (3, 1)])
def test_group_sizes(cuda_device, heads, kv_heads):
    c = Case(cuda_device, [(250, 5), (120, 17), (0, 2), (64, 40)], heads, kv_heads, seed=heads)
    c.check(*c.run())


@pytest.mark.parametrize("kind", ["random", "none", "all", "chain"])
@pytest.mark.parametrize("rows", ["no_prefix", "tile_edges", "wide"])
def test_any_mask(cuda_device, rows, kind):
    """Masks need not be trees; rows that see nothing give zeros."""
    c = Case(cuda_device, ROWS[rows], 4, 1, kind=kind, seed=3, extra_words=1)
    c.check(*c.run())


def test_large_logits(cuda_device):
    """The running maximum moves and rescales inside the nodes' own tiles too."""
    c = Case(cuda_device, [(900, 14), (90, 70)], 4, 1, seed=4, scale=8.0)
    c.check(*c.run())


@pytest.mark.parametrize("rows", ["ragged", "wide", "split", "idle_rows"])
def test_page_tables_and_device_plans(cuda_device, rows):
    c = Case(cuda_device, ROWS[rows], 8, 2, seed=5)
    first = c.run()
    c.check(*first)
    for kw in (dict(tables=True), dict(device_plan=True), dict(device_plan=True, tables=True), dict(trees=True),
               dict(device_plan=True, trees=True)):
        out, lse = c.run(**kw)
        c.check(out, lse)


@pytest.mark.parametrize("device_plan", [False, True])
def test_draft_rows_beside_trees(cuda_device, device_plan):
    """Rows of one token that read a draft table's pages in a batch with trees that read the block table's."""
    c = Case(cuda_device, [(500, 12), (95, 1), (30, 40), (0, 1), (2000, 1)], 8, 2, seed=27)
    draft = [False, True, False, True, True]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    cols = max(len(r) for r in c.pages)
    own = [r + [10 ** 6] * (cols - len(r)) for r in c.pages]
    none = [10 ** 6] * cols
    w = HolisticAttentionWrapper(torch.empty(1, device=cuda_device))
    w.set_page_tables(i32([0 if d else 1 for d in draft]).to(cuda_device),
                      i32([r if d else none for r, d in zip(own, draft)]).to(cuda_device),
                      i32([none if d else r for r, d in zip(own, draft)]).to(cuda_device))
    if device_plan:
        w.plan_device(i32(c.starts).to(cuda_device), i32(c.kv_indptr).to(cuda_device),
                      i32([(e - 1) % 16 + 1 for e in c.ends]).to(cuda_device), 8, 2, 128, 16, trees=True)
    else:
        w.plan_host(i32(c.starts), i32(c.kv_indptr), i32(c.ends), None, 8, 2, 128, 16, trees=True)
    c.check(*w.run(c.q.to(cuda_device), c.cache.to(cuda_device), tree_mask=c.mask, return_lse=True))
    assert w.device_status() == 0


@pytest.mark.parametrize("heads,kv_heads", [(4, 1), (16, 2), (10, 2)])
@pytest.mark.parametrize("rows", ["ragged", "wide", "split", "tile_edges"])
def test_device_plans_for_trees_hold_the_host_plans_items(cuda_device, rows, heads, kv_heads):
    c = Case(cuda_device, ROWS[rows], heads, kv_heads, seed=14)
    lists = []
    for device_plan in (False, True):
        w = c.plan(device_plan=device_plan, trees=True)
        torch.cuda.synchronize()
        words = w._int_workspace[256:].view(torch.int32).cpu()
        n, at = int(words[1]), int(words[5])
        items = words[at:at + 16 * n].view(n, 16)
        # (Where a group's partial rows lie and which descriptor it has is the planner's own.)
        lists.append((n, int(words[4]), int(words[15]), int(words[17]),
                      sorted(tuple(r[:12].tolist()) + (int(r[13]) >= 0, int(r[14]), int(r[15])) for r in items)))
    assert lists[0] == lists[1]


@pytest.mark.parametrize("heads,kv_heads", [(4, 1), (8, 2), (16, 4)])
@pytest.mark.parametrize("rows,sms", [([(4200, 17), (1432, 30), (50, 32)], 3), ([(9000, 17), (3060, 30), (50, 32)], 4),
                                      ([(5000, 33), (6001, 21), (8, 40)], 3)])
@pytest.mark.parametrize("kind", ["tree", "random"])
def test_items_whose_tiles_alternate_between_the_halves(cuda_device, rows, sms, heads, kv_heads, kind):
    """Long pieces of rows of one half; a group's last item may have one tile,
    so that the other half has none."""
    c = Case(cuda_device, rows, heads, kv_heads, kind=kind, seed=16)
    wrappers = [HolisticAttentionWrapper(torch.empty(1, device=cuda_device), num_sms=sms * kv_heads) for _ in range(2)]
    for w, device_plan in zip(wrappers, (False, True)):
        c.plan(wrapper=w, trees=True, device_plan=device_plan)
        torch.cuda.synchronize()
        words = w._int_workspace[256:].view(torch.int32).cpu()
        items = words[int(words[5]):int(words[5]) + 16 * int(words[1])].view(-1, 16)
        assert int(((items[:, 14] == 2) & (items[:, 15] == 1)).sum()) >= 2 * kv_heads
        c.check(*w.run(c.q.to(cuda_device), c.cache.to(cuda_device), tree_mask=c.mask, return_lse=True))
        assert w.device_status() == 0


def _short_rows_of_four_widths():
    rng = random.Random(21)
    return [(rng.randint(0, 500), rng.choice([4, 8, 12, 16])) for _ in range(48)]


def _long_rows_of_four_widths():
    rng = random.Random(403)
    return [(rng.randint(900, 9000), rng.choice([4, 8, 12, 16])) for _ in range(rng.randint(2, 30))]


@pytest.mark.parametrize("rows,sms", [(_short_rows_of_four_widths(), 1), (_short_rows_of_four_widths(), 2),
                                      (_long_rows_of_four_widths(), 11)])
def test_consecutive_items_of_other_widths(cuda_device, rows, sms):
    """A CTA's items have 16, 32, 48 and 64 columns in turn, whole and split ones."""
    c = Case(cuda_device, rows, 8, 2, seed=21)
    w = HolisticAttentionWrapper(torch.empty(1, device=cuda_device), num_sms=sms)
    c.plan(wrapper=w, trees=True)
    torch.cuda.synchronize()
    words = w._int_workspace[256:].view(torch.int32).cpu()
    items = words[int(words[5]):int(words[5]) + 16 * int(words[1])].view(-1, 16)
    columns = torch.maximum((items[:, 9] - items[:, 8] + 15) // 16 * 16, items[:, 15])
    assert columns.unique().tolist() == [16, 32, 48, 64] and items.shape[0] > 2 * sms
    assert bool((items[:, 11] > 1).any()) == (sms == 11)
    q, kv = c.q.to(cuda_device), c.cache.to(cuda_device)
    out, lse = w.run(q, kv, tree_mask=c.mask, return_lse=True)
    c.check(out, lse)
    for _ in range(20):
        o, l = w.run(q, kv, tree_mask=c.mask, return_lse=True)
        assert torch.equal(o, out) and torch.equal(l, lse)
    assert w.device_status() == 0


@pytest.mark.parametrize("rows,sms", [(_short_rows_of_four_widths(), 3), (_long_rows_of_four_widths(), 11),
                                      ([(4200, 17), (1432, 30), (50, 32), (300, 5)], 6)])
def test_waits_that_expire_at_different_places(cuda_device, built_library, rows, sms):
    c = Case(cuda_device, rows, 8, 2, seed=28)
    w = HolisticAttentionWrapper(torch.empty(1, device=cuda_device), num_sms=sms)
    q, kv = c.q.to(cuda_device), c.cache.to(cuda_device)

    def run():
        c.plan(wrapper=w, trees=True)
        w.clear_device_status()
        out, lse = w.run(q, kv, tree_mask=c.mask, return_lse=True)
        return out, lse, w.device_status()

    want = run()
    c.check(*want[:2])
    expired = 0
    for limit in (1, 500, 2000, 4000, 8000, 16000):
        for _ in range(5):
            _capi.check(built_library.aspire_set_wait_limit_ns(limit), "aspire_set_wait_limit_ns")
            try:
                first = run()
            finally:
                _capi.check(built_library.aspire_set_wait_limit_ns(0), "aspire_set_wait_limit_ns")
            assert first[2] in (0, _capi.STATUS_TIMEOUT)
            expired += first[2] != 0
            for got in ((first, run()) if first[2] == 0 else (run(),)):
                assert got[2] == 0 and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert expired


def test_a_plain_plan_is_made_again_for_trees_outside_captures(cuda_device):
    c = Case(cuda_device, [(300, 16), (40, 25)], 4, 1, seed=15)
    q, kv = c.q.to(cuda_device), c.cache.to(cuda_device)
    w = c.plan()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        out, lse = w.run(q, kv, tree_mask=c.mask, return_lse=True)
    assert w.plan_info.causal == 0
    g.replay()
    c.check(out, lse)
    c.check(*w.run(q, kv, tree_mask=c.mask, return_lse=True))
    assert w.plan_info.causal == 2
    g.replay()
    c.check(out, lse)
    plain = w.run(q, kv)  # and back
    assert w.plan_info.causal == 0 and torch.equal(plain.nan_to_num(9), c.plan().run(q, kv).nan_to_num(9))
    g.replay()
    c.check(out, lse)
    c.check(*w.run(q, kv, tree_mask=c.mask, return_lse=True))
    t = c.plan(trees=True)
    with pytest.raises(ValueError, match="tree_mask"):
        t.run(q, kv)
    with pytest.raises(ValueError, match="causal"):
        w.plan_host(torch.tensor(c.starts), torch.tensor(c.kv_indptr), torch.tensor(c.ends), w._kv_indices, 4, 1, 128, 16,
                    causal=True, trees=True)
    c.plan(wrapper=w)
    assert w.run(q, kv).shape == q.shape


def test_the_callers_arrays_may_change_before_the_first_run(cuda_device):
    c = Case(cuda_device, [(300, 16), (40, 25)], 4, 1, seed=17)
    w = HolisticAttentionWrapper(torch.empty(1, device=cuda_device))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    arrays = i32(c.starts), i32(c.kv_indptr), i32(c.ends)
    w.plan_host(*arrays, i32([p for r in c.pages for p in r]).to(cuda_device), 4, 1, 128, 16)
    for a in arrays:
        a.fill_(1)
    c.check(*w.run(c.q.to(cuda_device), c.cache.to(cuda_device), tree_mask=c.mask, return_lse=True))


def test_a_replay_that_finds_another_kind_of_plan_writes_nothing(cuda_device):
    c = Case(cuda_device, [(300, 16), (40, 25)], 4, 1, seed=18)
    q, kv = c.q.to(cuda_device), c.cache.to(cuda_device).nan_to_num(0)
    w = c.plan()
    w.run(q, kv)
    torch.cuda.synchronize()
    outs, graphs = [], []
    for mask in (None, c.mask):
        g = torch.cuda.CUDAGraph()
        out = torch.full_like(q, 7)
        with torch.cuda.graph(g):
            w.run(q, kv, out=out, tree_mask=mask)
        graphs.append(g), outs.append(out)
    w.run(q, kv, tree_mask=c.mask)  # now for trees
    graphs[0].replay()
    assert w.device_status() == 2 and bool((outs[0] == 7).all())  # BAD_PLAN
    w.clear_device_status()
    graphs[1].replay()
    assert w.device_status() == 0 and torch.equal(outs[1], w.run(q, kv, tree_mask=c.mask))
    outs[1].fill_(7)
    shape = w._kv_indices, 4, 1, 128, 16
    w.plan_host(torch.tensor(c.starts), torch.tensor(c.kv_indptr), torch.tensor(c.ends), *shape, causal=True)
    graphs[1].replay()
    assert w.device_status() == 2 and bool((outs[1] == 7).all())
    w.clear_device_status()
    graphs[0].replay()
    assert w.device_status() == 0 and torch.equal(outs[0], w.run(q, kv))


@pytest.mark.parametrize("device_plan", [False, True])
def test_little_float_workspace(cuda_device, device_plan):
    """Plans for trees split no further than the workspace has room for."""
    c = Case(cuda_device, [(3000, 9), (700, 33)], 8, 2, seed=19)
    for room in (0, 64 << 10, 600 << 10):
        w = HolisticAttentionWrapper(torch.empty(1, device=cuda_device), float_workspace_bytes=room)
        c.plan(wrapper=w, device_plan=device_plan, trees=True)
        c.check(*w.run(c.q.to(cuda_device), c.cache.to(cuda_device), tree_mask=c.mask, return_lse=True))
        assert w.device_status() == 0


def test_a_chain_is_the_causal_attention(cuda_device):
    c = Case(cuda_device, [(1200, 9), (60, 3), (400, 40)], 8, 2, kind="chain", seed=6)
    out, lse = c.run()
    w = HolisticAttentionWrapper(torch.empty(1, device=cuda_device))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    w.plan_host(i32(c.starts), i32(c.kv_indptr), i32(c.ends),
                i32([p for r in c.pages for p in r]).to(cuda_device), 8, 2, 128, 16, causal=True)
    c.check(*w.run(c.q.to(cuda_device), c.cache.to(cuda_device), return_lse=True))
    c.check(out, lse)


def test_strides_and_rows_behind_the_last(cuda_device):
    c = Case(cuda_device, [(140, 6), (31, 50)], 4, 2, seed=7, pad=5)
    w = c.plan()
    wide = torch.zeros(c.q.shape[0], 8, 256, dtype=torch.bfloat16, device=cuda_device)
    wide[:, 1::2, 64:192] = c.q.to(cuda_device)
    back = torch.full((c.q.shape[0], 4, 264), 7.0, dtype=torch.bfloat16, device=cuda_device)
    lse = torch.full((c.q.shape[0], 4), 7.0, device=cuda_device)
    out = w.run(wide[:, 1::2, 64:192], c.cache.to(cuda_device), tree_mask=c.mask, out=back[:, :, 8:136], lse=lse)
    c.check(out, lse)
    n = c.starts[-1]
    assert bool((back[n:] == 7).all()) and bool((lse[n:] == 7).all())
    assert bool((back[:n, :, :8] == 7).all()) and bool((back[:n, :, 136:] == 7).all())


def test_with_the_append_inside(cuda_device):
    c = Case(cuda_device, [(140, 6), (31, 5), (0, 3)], 8, 2, seed=8)
    n = c.starts[-1]
    k = torch.randn(n, 2, 128).to(torch.bfloat16)
    v = torch.randn(n, 2, 128).to(torch.bfloat16)
    cache = c.cache.to(cuda_device)
    w = c.plan()
    out, lse = w.run(c.q.to(cuda_device), cache, tree_mask=c.mask, return_lse=True,
                     append=(k.to(cuda_device), v.to(cuda_device)))
    for b, (a, m) in enumerate(c.rows):
        for i in range(m):
            page = c.pages[b][(a + i) // 16]
            c.cache[page, 0, (a + i) % 16] = k[c.starts[b] + i]
            c.cache[page, 1, (a + i) % 16] = v[c.starts[b] + i]
    c.check(out, lse)
    assert torch.equal(cache.cpu().nan_to_num(9), c.cache.nan_to_num(9))


def test_the_append_inside_larger_trees(cuda_device):
    """Rows of 65 to 127 packed queries are decode items of a plain plan, but not of one for trees."""
    c = Case(cuda_device, [(140, 20), (31, 5), (700, 31)], 8, 2, seed=25)
    n, q = c.starts[-1], c.q.to(cuda_device)
    k, v = (torch.randn(n, 2, 128, generator=torch.Generator().manual_seed(s)).to(torch.bfloat16) for s in (1, 2))
    cache = c.cache.to(cuda_device)
    w = c.plan()
    c.check(*w.run(q, cache, tree_mask=c.mask, return_lse=True))
    assert w.plan_info.causal == 2 and w.plan_info.num_items_prefill > 0
    for _ in range(2):
        out, lse = w.run(q, cache, tree_mask=c.mask, return_lse=True, append=(k.to(cuda_device), v.to(cuda_device)))
        assert w.plan_info.causal == 0 and w.plan_info.num_items_prefill == 0
    for b, (a, m) in enumerate(c.rows):
        for i in range(m):
            page = c.pages[b][(a + i) // 16]
            c.cache[page, 0, (a + i) % 16] = k[c.starts[b] + i]
            c.cache[page, 1, (a + i) % 16] = v[c.starts[b] + i]
    c.check(out, lse)
    assert torch.equal(cache.cpu().nan_to_num(9), c.cache.nan_to_num(9))
    c.check(*w.run(q, cache, tree_mask=c.mask, return_lse=True))
    assert w.plan_info.causal == 2 and w.device_status() == 0
    # More than a plain plan's decode items hold: refused, and the plan stays the caller's.
    c = Case(cuda_device, [(140, 32)], 8, 2, seed=26)
    w = c.plan()
    with pytest.raises(ValueError, match="append"):
        w.run(c.q.to(cuda_device), c.cache.to(cuda_device), tree_mask=c.mask, append=(k[:32].to(cuda_device), v[:32].to(cuda_device)))
    assert w.plan_info.causal == 0


def test_the_append_checks_its_operands(cuda_device):
    c = Case(cuda_device, [(140, 6), (31, 5)], 8, 2, seed=24)
    w, cache, n = c.plan(trees=True), c.cache.to(cuda_device), c.starts[-1]
    buf = torch.zeros(n, 12, 128, dtype=torch.bfloat16, device=cuda_device)  # a fused projection's output
    q, k, v = buf[:, :8], buf[:, 8:10], buf[:, 10:]
    part = cache[0, 0, :11]
    before = cache.clone()
    for kw, text in [(dict(append=(k, v), out=buf[:, 2:10]), "overlap"), (dict(append=(k, v), out=buf[:, 4:]), "overlap"),
                     (dict(append=(part, v)), "overlap"), (dict(append=(k, part)), "overlap"),
                     (dict(append=(k, None)), "both"), (dict(append=(k[:-1], v)), "k_new"), (dict(append=(k, v[:, :1])), "v_new"),
                     (dict(append=(k.float(), v)), "k_new"), (dict(append=(k, v.cpu())), "v_new"),
                     (dict(append=(k, v.detach().clone().requires_grad_())), "gradient")]:
        with pytest.raises(ValueError, match=text):
            w.run(q, cache, tree_mask=c.mask, **kw)
        assert torch.equal(cache.nan_to_num(9), before.nan_to_num(9))
    with pytest.raises(ValueError, match="gradient"):
        w.run(q.detach().clone().requires_grad_(), cache, tree_mask=c.mask, append=(k, v))
    version = cache._version
    w.run(q, cache, tree_mask=c.mask, append=(k, v), out=q)
    assert cache._version > version


def test_nodes_past_the_mask_are_hidden_under_device_plans(cuda_device):
    c = Case(cuda_device, [(50, 40), (20, 70)], 4, 1, kind="all", seed=9)
    c.mask = c.mask[:, :1].contiguous()
    for s in c.seen:
        s[:, 32:] = False
    c.check(*c.run(device_plan=True))


def test_bad_pages_are_reported(cuda_device):
    c = Case(cuda_device, [(50, 6)], 4, 1, seed=10)
    c.pages[0][1] = 10 ** 6
    w = c.plan()
    w.run(c.q.to(cuda_device), c.cache.to(cuda_device), tree_mask=c.mask)
    assert w.device_status() == 1


def test_replayed_with_other_masks_and_lengths(cuda_device):
    cases = [Case(cuda_device, rows, 8, 2, seed=s, extra_words=e) for s, (rows, e) in enumerate(
        [([(700, 12), (90, 3), (10, 40)], 0), ([(300, 30), (11, 20), (0, 5)], 1), ([(3, 1), (1500, 33), (0, 21)], 0)])]
    dev = cuda_device
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    starts, kvp, last = (torch.zeros(k, dtype=torch.int32, device=dev) for k in (4, 4, 3))
    flat = torch.zeros(400, dtype=torch.int32, device=dev)
    q = torch.zeros(55, 8, 128, dtype=torch.bfloat16, device=dev)
    cache = torch.zeros(200, 2, 16, 2, 128, dtype=torch.bfloat16, device=dev)
    mask = torch.zeros(55, 2, dtype=torch.int32, device=dev)
    w = HolisticAttentionWrapper(torch.empty(1, device=dev))

    def load(c):
        n = c.starts[-1]
        starts.copy_(i32(c.starts))
        kvp.copy_(i32(c.kv_indptr))
        last.copy_(i32([(e - 1) % 16 + 1 for e in c.ends]))
        ids = i32([p for r in c.pages for p in r])
        flat[:ids.numel()].copy_(ids)
        q[:n].copy_(c.q)
        cache[:c.cache.shape[0]].copy_(c.cache)
        mask[:n].copy_(c.mask)

    def step():
        w.plan_device(starts, kvp, last, 8, 2, 128, 16, paged_kv_indices=flat, trees=True)
        return w.run(q, cache, tree_mask=mask, return_lse=True)

    load(cases[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, lse = step()
    torch.cuda.synchronize()
    cases[0].check(out, lse)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = step()
    for c in cases[1:] + cases[:1]:
        load(c)
        g.replay()
        c.check(out, lse)
    assert w.device_status() == 0


def test_results_repeat_bit_by_bit(cuda_device):
    c = Case(cuda_device, [(2600, 12), (900, 50)], 8, 2, seed=12)
    out, lse = c.run()
    for _ in range(3):
        o, l = c.run()
        assert torch.equal(o, out) and torch.equal(l, lse)


def test_outputs_that_overlap_the_queries(cuda_device):
    c = Case(cuda_device, [(300, 5), (40, 20)], 4, 2, seed=23)
    w, kv, n = c.plan(trees=True), c.cache.to(cuda_device), c.starts[-1]
    buf = torch.zeros(n + 1, 12, 128, dtype=torch.bfloat16, device=cuda_device)
    flat = torch.zeros(2 * n * 4 * 128, dtype=torch.bfloat16, device=cuda_device)
    for q, out in [(buf[:-1, :4], buf[1:, :4]), (buf[:-1, :4], buf[:-1, 3:7]), (buf[:-1, :4], buf[:-1, :8:2]),
                   (buf[:-1, :8:2], buf[:-1, 2:10:2]), (buf[:-1, :4], buf.view(-1)[8:8 + 512 * n].view(n, 4, 128))]:
        before = buf.clone()
        with pytest.raises(ValueError, match="q itself"):
            w.run(q, kv, tree_mask=c.mask, out=out)
        assert torch.equal(buf, before)
    # Between one another's rows or heads, or itself.
    want = w.run(c.q.to(cuda_device), kv, tree_mask=c.mask)
    for q, out in [(buf[:-1, :4], buf[:-1, 4:8]), (buf[:-1, :8:2], buf[:-1, 1:8:2]), (buf[:-1, 2:10:2], buf[:-1, 2:10:2]),
                   (flat[:n * 512].view(4, n, 128).transpose(0, 1), flat[n * 512:].view(4, n, 128).transpose(0, 1))]:
        q.copy_(c.q)
        version = out._version
        assert torch.equal(w.run(q, kv, tree_mask=c.mask, out=out), want) and out._version > version
    for kw in (dict(out=torch.zeros_like(want, requires_grad=True)),
               dict(lse=torch.zeros(n, 4, device=cuda_device, requires_grad=True))):
        with pytest.raises(ValueError, match="requires a gradient"):
            w.run(c.q.to(cuda_device), kv, tree_mask=c.mask, **kw)
        with torch.no_grad():
            w.run(c.q.to(cuda_device), kv, tree_mask=c.mask, **kw)


@pytest.mark.parametrize("heads,kv_heads,nodes", [(4, 1, 5), (8, 2, 13), (5, 1, 7), (2, 1, 5)])
def test_neighbours_queries_leave_no_trace(cuda_device, heads, kv_heads, nodes):
    """The columns behind an item's rows hold the next row's queries, which must
    not decide when its own references move: small, large or not finite, the
    row's outputs keep their bits."""
    c = Case(cuda_device, [(1500, nodes), (700, nodes)], heads, kv_heads, seed=22, scale=4.0)
    w, kv = c.plan(trees=True), c.cache.to(cuda_device)
    runs = []
    for scale in (0.0, 1.0, 30.0, math.inf):
        q = c.q.to(cuda_device)
        q[nodes:] *= scale  # (inf and NaN in the last)
        runs.append(w.run(q, kv, tree_mask=c.mask, return_lse=True))
    c.check(*runs[1])
    for out, lse in runs:
        assert torch.equal(out[:nodes], runs[0][0][:nodes]) and torch.equal(lse[:nodes], runs[0][1][:nodes])


def test_refusals(cuda_device):
    c = Case(cuda_device, [(50, 40)], 4, 1, seed=13)
    q, kv = c.q.to(cuda_device), c.cache.to(cuda_device)
    w = c.plan()
    for mask in (c.mask.long(), c.mask[:, 0], c.mask[:-1], c.mask.cpu(), c.mask.repeat(1, 2)[:, ::2], c.mask[:, :0]):
        with pytest.raises(ValueError):
            w.run(q, kv, tree_mask=mask)
    with pytest.raises(ValueError, match="more queries"):
        w.run(q, kv, tree_mask=c.mask[:, :1].contiguous())
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    w.plan_host(i32(c.starts), i32(c.kv_indptr), i32(c.ends), i32(c.pages[0]).to(cuda_device), 4, 1, 128, 16, causal=True)
    with pytest.raises(ValueError, match="causal"):
        w.run(q, kv, tree_mask=c.mask)
    d = HolisticAttentionWrapper(torch.empty(1, device=cuda_device), jit_args=first_last_dump_jit_args())
    c.plan(wrapper=d)
    dump = torch.empty(4 * 2 * 96, dtype=torch.float16, device=cuda_device)
    with pytest.raises(ValueError, match="dump"):
        d.run(q, kv, dump, 4, 96, tree_mask=c.mask)


def test_outputs_that_overlap_are_refused(cuda_device):
    c = Case(cuda_device, [(30, 4)], 4, 1, seed=20)
    w, q, kv = c.plan(trees=True), c.q.to(cuda_device), c.cache.to(cuda_device)
    lse = torch.empty(4, 4, device=cuda_device)
    for kw in (dict(out=kv.view(-1)[:q.numel()].view(q.shape)), dict(lse=q.view(-1).view(torch.float32)[:16].view(4, 4)),
               dict(out=lse.new_empty(1024).view(torch.bfloat16).view(q.shape), lse=None)):
        if kw.get("lse", lse) is None:
            kw["lse"] = kw["out"].view(-1).view(torch.float32)[:16].view(4, 4)
        with pytest.raises(ValueError, match="overlap"):
            w.run(q, kv, tree_mask=c.mask, **kw)
    out = w.run(q, kv, tree_mask=c.mask)
    assert torch.equal(w.run(q, kv, tree_mask=c.mask, out=q), out)  # in place of the queries
