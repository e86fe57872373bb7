"""Block tables and slot maps from the rows' lengths (``build_step_tables``)
against the definition in Python: pages taken and given back, prefix sums,
positions, slots and masks, all of them integers."""

import random

import pytest
import torch

from aspire_b200.kv_ops import build_step_tables
import tree_reference as ref

pytestmark = pytest.mark.gpu


class Pool:
    """A pool of pages and the rows' tables, on the GPU and as lists."""

    def __init__(self, rng, dev, lengths, cols, page, spare, pad=0):
        rows = len(lengths)
        held = [-(-n // page) for n in lengths]
        ids = list(range(7, 7 + sum(held) + spare))
        rng.shuffle(ids)
        it = iter(ids)
        self.table = [[next(it) for _ in range(h)] + [-1] * (cols - h) for h in held]
        self.held = held
        self.count = spare
        self.free = [next(it) for _ in range(spare)] + [0] * sum(held)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        wide = torch.full((rows, cols + pad), 77, dtype=torch.int32, device=dev)
        if rows and cols:
            wide[:, :cols] = i32(self.table)
        self.wide, self.d_table = wide, wide[:, :cols]
        self.d_held, self.d_free, self.d_count = i32(held), i32(self.free), i32([spare])
        self.page, self.dev, self.status = page, dev, torch.zeros(1, dtype=torch.int32, device=dev)

    def step(self, lengths, new, tokens, parents=None, max_nodes=None, call=None):
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=self.dev)  # noqa: E731
        words = (max_nodes + 31) // 32 if parents is not None else 0
        exp, self.count, bad = ref.step_tables(lengths, new if new is not None else [0] * len(lengths), self.table,
                                               self.held, self.free, self.count, self.page, tokens, parents, words)
        self.status.zero_()
        got = (call or build_step_tables)(
            i32(lengths), i32(new) if new is not None else None, self.d_table, self.d_held, self.d_free, self.d_count,
            tokens=tokens, parents=i32(parents) if parents is not None else None, max_nodes=max_nodes,
            page_size=self.page, status=self.status)
        self.check(exp, got, bad)
        return got

    def check(self, exp, got, bad):
        for name, want in exp.items():
            have = getattr(got, name)
            if want is None:
                assert have is None
            else:
                assert have.cpu().tolist() == want, name
        assert got.slots.dtype == torch.int64
        assert self.d_table.cpu().tolist() == self.table
        assert self.d_held.cpu().tolist() == self.held
        assert int(self.d_count) == self.count
        assert self.d_free.cpu().tolist()[:self.count] == self.free[:self.count]
        assert int(self.status) == bad


@pytest.mark.parametrize("rows,page,most", [(1, 16, 5), (7, 16, 40), (64, 16, 9), (33, 1, 7), (40, 7, 100),
                                            (1500, 16, 3), (3, 16, 5000)])
def test_chain_steps_take_and_give_back(cuda_device, rows, page, most):
    rng = random.Random(rows * 100 + page)
    lengths = [rng.choice([0, 1, page - 1, page, page + 1, rng.randint(0, 300)]) for _ in range(rows)]
    cols = -(-(max(lengths) + 4 * most) // page) + 1
    pool = Pool(rng, cuda_device, lengths, cols, page, rows * (-(-4 * most // page) + 2), pad=3)
    for _ in range(4):
        new = [rng.choice([0, 1, most, rng.randint(0, most)]) for _ in range(rows)]
        pool.step(lengths, new, sum(new) + rng.choice([0, 5]))
        # Some of the tokens stay, as after a verification.
        lengths = [a + rng.randint(0, n) for a, n in zip(lengths, new)]
        if rng.random() < 0.5:
            pool.step(lengths, None, 0)
    # Finished rows give everything back; the columns behind the table stay as they were.
    pool.step([0] * rows, None, 0)
    assert all(v == -1 for r in pool.table for v in r)
    assert bool((pool.wide[:, cols:] == 77).all())


@pytest.mark.parametrize("rows,nodes", [(1, 1), (1, 32), (5, 33), (64, 48), (9, 100), (3, 300)])
def test_trees(cuda_device, rows, nodes):
    rng = random.Random(nodes)
    lengths = [rng.randint(0, 200) for _ in range(rows)]
    new = [nodes] + [rng.choice([0, rng.randint(1, nodes)]) for _ in range(rows - 1)]
    pool = Pool(rng, cuda_device, lengths, 64, 16, rows * (nodes // 16 + 2))
    parents = [p for n in new for p in (ref.random_parents(rng, n, 9) if n else [])] + [0, 1, 2]
    pool.step(lengths, new, sum(new) + 3, parents, nodes)
    pool.step(lengths, None, 0)


def test_giving_back_leaves_the_stack_as_it_was(cuda_device):
    rng = random.Random(1)
    lengths = [rng.randint(0, 100) for _ in range(20)]
    pool = Pool(rng, cuda_device, lengths, 40, 16, 200)
    before = [t.clone() for t in (pool.d_table, pool.d_held, pool.d_free[:200], pool.d_count)]
    pool.step(lengths, [rng.randint(0, 70) for _ in range(20)], 20 * 70)
    pool.step(lengths, None, 0)
    for a, b in zip(before, (pool.d_table, pool.d_held, pool.d_free[:200], pool.d_count)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("spare", [0, 1, 3, 6])
def test_rows_are_served_until_the_pages_run_out(cuda_device, spare):
    rng = random.Random(spare)
    lengths = [16, 15, 16, 40, 32, 3]
    pool = Pool(rng, cuda_device, lengths, 8, 16, spare)
    pool.step(lengths, [1, 1, 20, 30, 0, 2], 60)


def test_pages_given_back_serve_the_same_call(cuda_device):
    rng = random.Random(5)
    pool = Pool(rng, cuda_device, [160, 16, 16], 12, 16, 0)
    pool.step([5, 16, 16], [3, 60, 90], 200)


def test_rows_that_do_not_fit(cuda_device):
    rng = random.Random(6)
    lengths = [30, 30, 30]
    pool = Pool(rng, cuda_device, lengths, 4, 16, 20)
    pool.step(lengths, [35, 34, 2], 71)  # 65 tokens need a fifth column
    # A tree of more nodes than its masks have bits, beside one that fits.
    pool = Pool(rng, cuda_device, lengths, 8, 16, 20)
    pool.step(lengths, [33, 32, 1], 66, [p for n in (33, 32, 1) for p in ref.random_parents(rng, n)], 32)


def test_parents_that_are_no_earlier_nodes(cuda_device):
    rng = random.Random(7)
    pool = Pool(rng, cuda_device, [4, 4], 4, 16, 4)
    pool.step([4, 4], [4, 3], 7, [-1, 1, 0, 9, 0, -5, 1], 8)


def test_token_buffers_that_are_too_short(cuda_device):
    rng = random.Random(8)
    pool = Pool(rng, cuda_device, [4, 4], 4, 16, 4)
    pool.step([4, 4], [4, 3], 5)


def test_no_rows_and_no_tokens(cuda_device):
    rng = random.Random(9)
    pool = Pool(rng, cuda_device, [], 4, 16, 4)
    got = pool.step([], [], 3, [0, 0, 0], 40)
    assert got.tree_mask.shape == (3, 2)
    pool = Pool(rng, cuda_device, [3], 4, 16, 4)
    pool.step([3], [0], 0, [], 4)


def test_negative_entries_count_as_zero(cuda_device):
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda_device)  # noqa: E731
    status = i32(0)
    table = torch.full((2, 3), -1, dtype=torch.int32, device=cuda_device)
    got = build_step_tables(i32(-4, 3), i32(2, -9), table, i32(0, -1), i32(5, 6, 7), i32(3), tokens=2, status=status)
    assert got.kv_len.tolist() == [2, 3] and got.qo_indptr.tolist() == [0, 2, 2]
    assert got.slots.tolist() == [6 * 16, 6 * 16 + 1] and table.tolist() == [[6, -1, -1], [7, -1, -1]]
    assert int(status) == 4


def test_a_count_past_the_capacity_is_bounded(cuda_device):
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda_device)  # noqa: E731
    status, count = i32(0), i32(9)
    table = torch.tensor([[1, 2]], dtype=torch.int32, device=cuda_device)
    build_step_tables(i32(0), None, table, i32(2), i32(5, 6, 7), count, tokens=0, status=status)
    assert int(count) == 3 and int(status) == 4 and table.tolist() == [[-1, -1]]


def test_captured_and_replayed_on_another_stream(cuda_device):
    rng = random.Random(11)
    lengths = [rng.randint(0, 60) for _ in range(6)]
    pool = Pool(rng, cuda_device, lengths, 12, 16, 40)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda_device)  # noqa: E731
    new = [rng.randint(1, 9) for _ in range(6)]
    parents = [p for n in new for p in ref.random_parents(rng, n)]
    d_len, d_new = i32(lengths), i32(new)
    d_par = torch.nn.functional.pad(i32(parents), (0, 60 - len(parents)))
    args = (d_len, d_new, pool.d_table, pool.d_held, pool.d_free, pool.d_count)
    state = [t.clone() for t in args[2:]]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        build_step_tables(*args, tokens=60, parents=d_par, max_nodes=9, status=pool.status)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = build_step_tables(*args, tokens=60, parents=d_par, max_nodes=9, status=pool.status)
    for t, s in zip(args[2:], state):
        t.copy_(s)
    for _ in range(3):
        exp, pool.count, bad = ref.step_tables(lengths, new, pool.table, pool.held, pool.free, pool.count, 16, 60,
                                               parents, 1)
        g.replay()
        torch.cuda.synchronize()
        pool.check(exp, got, bad)
        lengths = [a + 3 for a in lengths]
        d_len.copy_(i32(lengths))
