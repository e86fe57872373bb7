"""The accepted path and the move of its keys and values (``accept_tree``)
against the definition in Python."""

import random

import pytest
import torch

from aspire_b200.tree import accept_tree
import tree_reference as ref

pytestmark = pytest.mark.gpu


def _case(rng, sizes, most, page, cols, tokens_of=6):
    """Few token values, so that walks go deep and siblings repeat."""
    rows = []
    for n in sizes:
        parents = ref.random_parents(rng, n, 4) if n else []
        rows.append((parents, [rng.randrange(tokens_of) for _ in range(n)], [rng.randrange(tokens_of) for _ in range(n)]))
    lengths = [rng.randint(0, cols * page - max(n, 1)) for n in sizes]
    paths = [ref.walk(t, p, w, most) for p, t, w in rows]
    return rows, lengths, paths


def _run(dev, rng, sizes, most, page=16, heads=2, dim=128, layers=3, dtype=torch.bfloat16, cols=5, tokens_of=6,
         total_pad=0):
    rows, lengths, paths = _case(rng, sizes, most, page, cols, tokens_of)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    flat = lambda k: i32([v for r in rows for v in r[k]] + [1] * total_pad)  # noqa: E731
    pages = len(sizes) * cols + 2
    order = list(range(pages))
    rng.shuffle(order)
    table = [order[b * cols:(b + 1) * cols] for b in range(len(sizes))]
    caches = [torch.randn(pages, 2, page, heads, dim, device=dev).to(dtype) for _ in range(layers)]
    exp = [c.clone() for c in caches]
    place = lambda b, i: (table[b][i // page], i % page)  # noqa: E731
    for c in exp:
        src = c.clone()
        for b, path in enumerate(paths):
            for d, node in enumerate(path):
                (sp, so), (dp, do) = place(b, lengths[b] + node), place(b, lengths[b] + d)
                c[dp, :, do] = src[sp, :, so]
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    a = accept_tree(flat(1), flat(0), flat(2), i32(ref.indptr(sizes)), i32(lengths), most, caches=caches,
                    block_table=torch.tensor(table, dtype=torch.int32, device=dev) if layers else None, status=status)
    assert a.count.tolist() == [len(p) for p in paths]
    assert a.path.tolist() == [p + [-1] * (most - len(p)) for p in paths]
    assert a.tokens.tolist() == [[rows[b][2][n] for n in p] + [-1] * (most - len(p)) for b, p in enumerate(paths)]
    assert a.lengths.tolist() == [n + len(p) for n, p in zip(lengths, paths)]
    for c, e in zip(caches, exp):
        assert torch.equal(c, e)
    assert int(status) == 0
    return paths


@pytest.mark.parametrize("sizes,most", [([1], 1), ([9], 5), ([0, 1, 2, 33, 64, 100, 7], 12), ([40] * 70, 64),
                                        ([1500], 64)])
def test_walks_and_moves(cuda_device, sizes, most):
    _run(cuda_device, random.Random(len(sizes) * 100 + most), sizes, most, cols=100 if max(sizes) > 1000 else 9)


@pytest.mark.parametrize("page,heads,dim,dtype", [(16, 8, 128, torch.bfloat16), (1, 1, 64, torch.float16),
                                                  (7, 3, 8, torch.float32), (32, 1, 16, torch.uint8)])
def test_cache_layouts(cuda_device, page, heads, dim, dtype):
    rng = random.Random(page)
    sizes = [rng.randint(0, 30) for _ in range(12)]
    if dtype == torch.uint8:
        torch.manual_seed(0)
    _run(cuda_device, rng, sizes, 8, page=page, heads=heads, dim=dim, dtype=dtype, cols=-(-64 // page), tokens_of=2)


@pytest.mark.parametrize("layers", [0, 1, 130])
def test_layers(cuda_device, layers):
    _run(cuda_device, random.Random(layers), [12, 0, 30, 5], 9, layers=layers, heads=1, tokens_of=2, total_pad=3)


def test_a_path_that_moves_over_its_own_places(cuda_device):
    """node_1 = 2 moves to place 1 and node_2 = 3 to place 2, where node_1 lay."""
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda_device)  # noqa: E731
    n = 40
    parents = [-1, 0] + list(range(0, 1)) + list(range(2, n - 1))
    tokens = [0, 5] + [7] * (n - 2)
    cache = torch.randn(4, 2, 16, 2, 128, device=cuda_device).to(torch.bfloat16)
    want = cache.clone()
    order = [2, 0, 3, 1]
    for d in range(1, 30):
        want[order[d // 16], :, d % 16] = cache[order[(d + 1) // 16], :, (d + 1) % 16]
    a = accept_tree(i32(tokens), i32(parents), i32([7] * n), i32([0, n]), i32([0]), 30, caches=[cache],
                    block_table=i32([order]))
    assert a.path[0].tolist() == [0] + list(range(2, 31))
    assert torch.equal(cache, want)


def test_places_without_a_page_are_not_moved(cuda_device):
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda_device)  # noqa: E731
    status = i32([0])
    cache = torch.randn(4, 2, 16, 1, 128, device=cuda_device).to(torch.bfloat16)
    before = cache.clone()
    # Row 0's second page is no page of the cache, row 1's place lies behind its table, row 2's indptr is wrong.
    a = accept_tree(i32([1, 2, 3, 1, 2, 3]), i32([-1, 0, 0, -1, 0, 0]), i32([3, 0, 0, 3, 0, 0]), i32([0, 3, 6, 9]),
                    i32([14, 31, 0]), 4, caches=[cache], block_table=i32([[0, 9], [1, 2], [3, 3]]), status=status)
    assert a.count.tolist() == [2, 2, 0]
    assert torch.equal(cache, before)
    assert int(status) == 5


def test_only_nodes_with_keys_in_the_cache_are_walked(cuda_device):
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda_device)  # noqa: E731
    status = i32([0])
    cache = torch.randn(6, 2, 16, 1, 128, device=cuda_device).to(torch.bfloat16)
    before = cache.clone()
    # Rows 0 and 1: no page at their second node's place (no page of the cache; behind the table).  Row 2 got no
    # pages, row 3 has all that it needs, row 4 is row 3 with a key less.
    args = (i32([1, 2, 3] * 5), i32([-1, 0, 0] * 5), i32([3, 7, 8] * 5), i32([0, 3, 6, 9, 12, 15]),
            i32([14, 31, 6, 2, 2]), 4)
    table = i32([[0, 9], [1, 2], [3, 3], [4, -1], [5, -1]])
    a = accept_tree(*args, caches=[cache], block_table=table, kv_len=i32([17, 34, 0, 5, 4]), status=status)
    assert a.count.tolist() == [1, 1, 0, 2, 1]
    assert a.path.tolist() == [[0, -1, -1, -1]] * 2 + [[-1] * 4, [0, 2, -1, -1], [0, -1, -1, -1]]
    assert a.tokens.tolist() == [[3, -1, -1, -1]] * 2 + [[-1] * 4, [3, 8, -1, -1], [3, -1, -1, -1]]
    assert a.lengths.tolist() == [15, 32, 6, 4, 3]
    before[4, :, 3] = before[4, :, 4]
    assert torch.equal(cache, before)
    assert int(status) == 1
    # The walk alone knows no pages.
    a = accept_tree(*args, kv_len=i32([17, 34, 0, 5, -3]))
    assert a.count.tolist() == [2, 2, 0, 2, 0]
    for bad in (i32([1] * 4), i32([1] * 5).long(), i32([1] * 5).cpu()):
        with pytest.raises(ValueError, match="kv_len"):
            accept_tree(*args, kv_len=bad)


def test_a_node_without_a_choice_is_not_committed(cuda_device):
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda_device)  # noqa: E731
    # Drafts of -1 are padding: 0 -> 2 -> 3 -> 4 in each row, without a choice after node 0, 2 and 4, and with all.
    tokens, parents = [1, -1, 5, 6, -1], [-1, 0, 0, 2, 3]
    targets = [[-1, 0, 6, -7, 9], [5, 0, -1, 9, 9], [5, 0, 6, -(2 ** 31), 9], [5, 0, 6, 9, -1]]
    cache = torch.randn(4, 2, 16, 1, 128, device=cuda_device).to(torch.bfloat16)
    want = cache.clone()
    for b, moved in enumerate([[], [], [2], [2, 3]]):
        for d, node in enumerate(moved):
            want[b, :, 3 + d + 1] = cache[b, :, 3 + node]
    status = i32([0])
    a = accept_tree(i32(tokens * 4), i32(parents * 4), i32([v for r in targets for v in r]), i32([0, 5, 10, 15, 20]),
                    i32([3] * 4), 5, caches=[cache], block_table=i32([[0], [1], [2], [3]]), status=status)
    assert a.path.tolist() == [[-1] * 5, [0] + [-1] * 4, [0, 2, -1, -1, -1], [0, 2, 3, -1, -1]]
    assert a.tokens.tolist() == [[-1] * 5, [5] + [-1] * 4, [5, 6, -1, -1, -1], [5, 6, 9, -1, -1]]
    assert a.count.tolist() == [0, 1, 2, 3] and a.lengths.tolist() == [3, 4, 5, 6]
    assert torch.equal(cache, want)
    assert int(status) == 32
    # The path's end comes first.
    a = accept_tree(i32(tokens), i32(parents), i32(targets[2]), i32([0, 5]), i32([3]), 2, status=status.zero_())
    assert a.path[0].tolist() == [0, 2] and int(status) == 0


def test_captured_and_replayed(cuda_device):
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda_device)  # noqa: E731
    tokens, parents, targets = i32([1, 2, 3, 4]), i32([-1, 0, 0, 2]), i32([3, 0, 4, 0])
    at, lengths, table = i32([0, 4]), i32([2]), i32([[1, 0]])
    cache = torch.randn(2, 2, 16, 1, 128, device=cuda_device).to(torch.bfloat16)
    first = cache.clone()
    args = (tokens, parents, targets, at, lengths, 3)
    accept_tree(*args, caches=[cache], block_table=table)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a = accept_tree(*args, caches=[cache], block_table=table)
    for want in ([0, 2, 3], [0, 1, -1]):
        cache.copy_(first)
        g.replay()
        assert a.path[0].tolist() == want
        exp = first.clone()
        if want[1] == 2:
            exp[1, :, 3], exp[1, :, 4] = first[1, :, 4], first[1, :, 5]
        assert torch.equal(cache, exp)
        targets.copy_(i32([2, 0, 4, 0]))
