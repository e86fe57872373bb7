"""Steps of tree speculation with all their operators, one after the other and
as one captured graph, on a model small enough to be followed in 64 bits: two
layers whose queries, keys and values are tables over the vocabulary, so that
the cache does not depend on how the committed tokens came to be."""

import random

import pytest
import torch

from aspire_b200.attention import HolisticAttentionWrapper
from aspire_b200.kv_ops import build_step_tables, qkv_prologue
from aspire_b200.logits import pick_tokens
from aspire_b200.tree import accept_tree
import tree_reference as ref

pytestmark = pytest.mark.gpu

VOCAB, HEADS, KV, LAYERS, COLS, MOST = 13, 4, 2, 2, 12, 6
TREE = [-1, 0, 0, 0, 0, 0, 1, 1, 2, 2, 3, 5, 7, 7, 12]


class Model:
    def __init__(self, dev, rows, seed):
        g = torch.Generator().manual_seed(seed)
        table = lambda h: torch.randn(VOCAB, h, 128, generator=g).to(torch.bfloat16).to(dev)  # noqa: E731
        self.q, self.k, self.v = ([table(h) for _ in range(LAYERS)] for h in (HEADS, KV, KV))
        self.out = torch.randn(LAYERS * HEADS * 128, VOCAB, generator=g, dtype=torch.float64).to(dev)
        self.norms = [(torch.rand(128, generator=g) + 0.5).to(torch.bfloat16).to(dev) for _ in range(2)]
        order = list(range(rows * COLS + 3))
        random.Random(seed).shuffle(order)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        self.free, self.count = i32(order), i32([len(order)])
        self.table, self.held = i32([[-1] * COLS] * rows), i32([0] * rows)
        self.pool = (self.table, self.held, self.free, self.count)
        self.modes = i32([1] * rows)
        self.caches = [torch.zeros(len(order), 2, 16, KV, 128, dtype=torch.bfloat16, device=dev) for _ in range(LAYERS)]
        self.wrapper = HolisticAttentionWrapper(torch.empty(1, device=dev))
        self.wrapper.set_page_tables(self.modes, self.table, self.table)

    def keys(self, l, tokens, t, **where):
        ids = tokens.long()
        return qkv_prologue(self.q[l][ids], self.k[l][ids], self.v[l][ids], t.qo_indptr, where.get("offsets"),
                            self.caches[l], None, t.kv_indptr, t.last_page_len, q_norm_weight=self.norms[0],
                            k_norm_weight=self.norms[1], page_tables=(self.modes, self.table, self.table),
                            positions=where.get("positions"))

    def chain(self, tokens, new, zeros):
        """The rows' tokens into empty tables: rotated queries by layer."""
        t = build_step_tables(zeros, new, *self.pool, tokens=tokens.shape[0])
        return [self.keys(l, tokens, t, offsets=zeros) for l in range(LAYERS)]

    def step(self, tokens, new, parents, lengths, history, frequency, status):
        t = build_step_tables(lengths, new, *self.pool, tokens=tokens.shape[0], parents=parents, max_nodes=len(TREE),
                              status=status)
        self.wrapper.plan_device(t.qo_indptr, t.kv_indptr, t.last_page_len, HEADS, KV, 128, 16, trees=True)
        outs = []
        for l in range(LAYERS):
            q = self.keys(l, tokens, t, positions=t.positions)
            outs.append(self.wrapper.run(q, self.caches[l], tree_mask=t.tree_mask, out=torch.zeros_like(q)))
        logits = (torch.cat([o.flatten(1) for o in outs], 1).double() @ self.out).float()
        targets = pick_tokens(logits, history=history, history_len=lengths, indptr=t.qo_indptr, tokens=tokens,
                              tree_mask=t.tree_mask, frequency=frequency, status=status)
        a = accept_tree(tokens, parents, targets, t.qo_indptr, lengths, MOST, caches=self.caches,
                        block_table=self.table, status=status)
        build_step_tables(a.lengths, None, *self.pool, tokens=0, status=status)
        return t, outs, logits, targets, a


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("prompts,seed", [([5, 37, 0], 0), ([16], 1), ([31, 1, 15, 48, 17], 2)])
def test_steps(cuda_device, prompts, seed, captured):
    dev, rows = cuda_device, len(prompts)
    rng = random.Random(seed)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    m = Model(dev, rows, seed)
    n_steps, T = 8, rows * len(TREE) + 4
    committed = [[rng.randrange(VOCAB) for _ in range(n)] for n in prompts]
    roots = [rng.randrange(VOCAB) for _ in prompts]
    if sum(prompts):
        m.chain(i32([v for c in committed for v in c]), i32(prompts), i32([0] * rows))
    frequency = torch.rand(rows, generator=torch.Generator().manual_seed(seed)).to(dev)
    tokens, parents = i32([0] * T), i32([-1] * T)
    new, lengths, status = i32([1] * rows), i32(prompts), i32([0])
    history = i32([[0] * (16 * COLS)] * rows)
    args = (tokens, new, parents, lengths, history, frequency, status)
    graph = None
    seen_out = [[{} for _ in prompts] for _ in range(LAYERS)]  # outputs at committed places
    longest = 0
    for step in range(n_steps):
        # A row may sit a step out; its tree may be its root alone.
        sizes = [0 if rows > 1 and rng.random() < 0.15 else rng.choice([1, len(TREE), len(TREE), 9]) for _ in prompts]
        trees = [[roots[b]] + [0] * (n - 1) if n else [] for b, n in enumerate(sizes)]
        for tree in trees:
            for i in range(1, len(tree)):  # siblings differ
                tree[i] = rng.choice([v for v in range(VOCAB) if v not in [
                    tree[j] for j in range(1, i) if TREE[j] == TREE[i]]])
        start = ref.indptr(sizes)
        pad = T - start[-1]
        tokens.copy_(i32([v for tree in trees for v in tree] + [rng.randrange(VOCAB) for _ in range(pad)]))
        parents.copy_(i32([p for n in sizes for p in TREE[:n]] + [-1] * pad))
        new.copy_(i32(sizes))
        lengths.copy_(i32([len(c) for c in committed]))
        history.copy_(i32([c + [0] * (16 * COLS - len(c)) for c in committed]))
        if not captured:
            t, outs, logits, targets, a = m.step(*args)
        else:
            if graph is None:  # (loading what the step needs: rows without tokens change nothing)
                new.zero_()
                m.step(*args)
                new.copy_(i32(sizes))
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    t, outs, logits, targets, a = m.step(*args)
            graph.replay()
        assert int(status) == 0 and m.wrapper.device_status() == 0
        assert t.qo_indptr.tolist() == start
        # The targets, from the logits that were there.
        row_of = [b for b, n in enumerate(sizes) for _ in range(n)] + [-1] * pad
        paths = [[tree[j] for j in p] for tree, n in zip(trees, sizes) for p in ref.ancestors(TREE[:n])]
        x, _, _ = ref.adjust(logits.cpu(), row_of, committed, [0] * rows, paths + [[]] * pad, None, frequency.cpu(),
                             None, None, None)
        want = ref.pick(x, row_of)
        assert targets.tolist() == want
        for b, tree in enumerate(trees):
            path = ref.walk(tree, TREE[:len(tree)], want[start[b]:start[b + 1]], MOST)
            assert a.path[b].tolist() == path + [-1] * (MOST - len(path))
            for node in path:
                for l in range(LAYERS):
                    seen_out[l][b][len(committed[b])] = outs[l][start[b] + node].clone()
                committed[b].append(tree[node])
                roots[b] = want[start[b] + node]
            longest = max(longest, len(path))
        assert a.lengths.tolist() == [len(c) for c in committed]
        pages = [-(-len(c) // 16) for c in committed]
        assert m.held.tolist() == pages and int(m.count) == rows * COLS + 3 - sum(pages)
    assert longest > 1
    held = [m.table[b, :p].tolist() for b, p in enumerate(pages)]
    assert len({p for r in held for p in r} | set(m.free[:int(m.count)].tolist())) == rows * COLS + 3

    # The same tokens as one chain: the same keys and values, bit for bit, and
    # every committed node's attention within its bound.
    c = Model(dev, rows, seed)
    sizes = [len(r) for r in committed]
    q = c.chain(i32([v for r in committed for v in r]), i32(sizes), i32([0] * rows))
    chain_pages = [c.table[b, :p].tolist() for b, p in enumerate(pages)]
    start = ref.indptr(sizes)
    for l in range(LAYERS):
        for b, n in enumerate(sizes):
            ours = m.caches[l][i32(held[b]).long()].transpose(1, 2).flatten(0, 1)[:n]
            assert torch.equal(ours, c.caches[l][i32(chain_pages[b]).long()].transpose(1, 2).flatten(0, 1)[:n])
        exp, _, bound, _ = ref.tree_attention(q[l].cpu(), c.caches[l].cpu(), chain_pages, start, sizes,
                                              [torch.ones(n, n, dtype=torch.bool).tril() for n in sizes])
        for b, by_place in enumerate(seen_out[l]):
            for place, out in by_place.items():
                t = start[b] + place
                assert bool(((out.double().cpu() - exp[t]).abs() <= bound[t]).all()), (l, b, place)


@pytest.mark.parametrize("captured", [False, True])
def test_a_step_in_which_the_pages_run_out(cuda_device, captured):
    """The last row's pages are not there at first: it commits nothing, keeps
    its length and its pages, and is served once another row has left."""
    dev, prompts, nodes = cuda_device, [20, 30, 13], len(TREE)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    rng = random.Random(9)
    m = Model(dev, 3, 9)
    committed = [[rng.randrange(VOCAB) for _ in range(n)] for n in prompts]
    m.chain(i32([v for c in committed for v in c]), i32(prompts), i32([0] * 3))  # 2, 2 and 1 pages
    m.count.fill_(2)  # 3, 3 and 2 pages are needed for the trees
    trees = [[rng.randrange(VOCAB)] + [i % VOCAB for i in range(1, nodes)] for _ in prompts]
    tokens, parents = i32([v for t in trees for v in t]), i32(TREE * 3)
    lengths, new, status = i32(prompts), i32([nodes] * 3), i32([0])
    frequency, history = torch.zeros(3, device=dev), i32([c + [0] * (16 * COLS - len(c)) for c in committed])

    def step():
        t = build_step_tables(lengths, new, *m.pool, tokens=3 * nodes, parents=parents, max_nodes=nodes, status=status)
        m.wrapper.plan_device(t.qo_indptr, t.kv_indptr, t.last_page_len, HEADS, KV, 128, 16, trees=True)
        outs = []
        for l in range(LAYERS):
            q = m.keys(l, tokens, t, positions=t.positions)
            outs.append(m.wrapper.run(q, m.caches[l], tree_mask=t.tree_mask))
        logits = (torch.cat([o.flatten(1) for o in outs], 1).double() @ m.out).float()
        targets = pick_tokens(logits, history=history, history_len=lengths, indptr=t.qo_indptr, tokens=tokens,
                              tree_mask=t.tree_mask, frequency=frequency, status=status)
        a = accept_tree(tokens, parents, targets, t.qo_indptr, lengths, MOST, caches=m.caches, block_table=m.table,
                        kv_len=t.kv_len, status=status)
        build_step_tables(a.lengths, None, *m.pool, tokens=0, status=status)
        return t, targets, a

    graph = None
    if captured:
        new.zero_()
        step()
        new.fill_(nodes)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            t, targets, a = step()

    def check(served, bits):
        nonlocal t, targets, a
        if captured:
            graph.replay()
        else:
            t, targets, a = step()
        assert int(status) == bits and m.wrapper.device_status() == 0
        starts, want = t.qo_indptr.tolist(), targets.tolist()
        for b in range(3):
            tree = trees[b][:starts[b + 1] - starts[b]]
            path = ref.walk(tree, TREE[:len(tree)], want[starts[b]:starts[b + 1]], MOST) if b in served else []
            assert a.path[b].tolist() == path + [-1] * (MOST - len(path))
            assert a.lengths[b] == len(committed[b]) + len(path)
            committed[b] += [tree[j] for j in path]
        assert m.held.tolist() == [-(-len(c) // 16) for c in committed]

    if not captured:
        t = targets = a = None
    first = m.caches[0][m.table[2, 0].long()].clone()
    check({0, 1}, 16)
    assert len(committed[2]) == 13 and torch.equal(m.caches[0][m.table[2, 0].long()], first)
    # Row 0 leaves.
    status.zero_()
    committed[0] = []
    lengths.copy_(i32([0] + [len(c) for c in committed[1:]]))
    new.copy_(i32([0, 1, nodes]))
    trees = [trees[0], [rng.randrange(VOCAB)], trees[2]]
    tokens.copy_(i32(trees[1] + trees[2] + [0] * (2 * nodes - 1)))
    parents.copy_(i32([-1] + TREE + [-1] * (2 * nodes - 1)))
    history.copy_(i32([c + [0] * (16 * COLS - len(c)) for c in committed]))
    check({0, 1, 2}, 0)
    assert len(committed[2]) > 13

    # The same keys and values as the tokens' own chain, bit for bit.
    c = Model(dev, 3, 9)
    c.chain(i32([v for r in committed for v in r]), i32([len(r) for r in committed]), i32([0] * 3))
    for l in range(LAYERS):
        for b, r in enumerate(committed):
            ours, chain = ((x.caches[l][x.table[b, :-(-len(r) // 16)].long()].transpose(1, 2).flatten(0, 1)[:len(r)])
                           for x in (m, c))
            assert torch.equal(ours, chain)
