"""Penalties, biases and grammar masks on logits against the definition: in 64
bits with the bound of the fp32 roundings, and the best token against the same
formula in fp32, step by step."""

import math
import random

import pytest
import torch

from aspire_b200 import _capi
from aspire_b200.logits import adjust_logits, pick_tokens
import tree_reference as ref

pytestmark = pytest.mark.gpu


def _pack(allowed):
    t, v = allowed.shape
    words = (v + 31) // 32
    bits = torch.zeros(t, words * 32, dtype=torch.int64)
    bits[:, :v] = allowed.long()
    w = (bits.view(t, words, 32) << torch.arange(32)).sum(2)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)


class Case:
    def __init__(self, seed, sizes, vocab, dtype, hist=50, bias=0, allowed=False, tree=True, path=True, prompt=True,
                 terms=("repetition", "frequency", "presence"), pad=0, row_pad=0, dense=False):
        rng = random.Random(seed)
        g = torch.Generator().manual_seed(seed)
        rows, total = len(sizes), sum(sizes)
        t = total + pad
        self.base = (torch.randn(t, vocab + row_pad, generator=g) * 3).to(dtype)
        self.logits = self.base[:, :vocab]
        span = max(2, vocab // 4) if not dense else 5
        ident = lambda: rng.choice([rng.randrange(min(span, vocab)), rng.randrange(vocab), vocab - 1, 0])  # noqa: E731
        self.history = [[ident() for _ in range(rng.choice([0, 1, hist, rng.randint(0, hist)]))] for _ in range(rows)]
        self.prompts = [rng.choice([0, len(h) // 2, len(h)]) if prompt else 0 for h in self.history]
        self.row_of = [b for b, n in enumerate(sizes) for _ in range(n)] + [-1] * pad
        self.tokens = [ident() for _ in range(t)]
        paths = [p for n in sizes for p in (ref.ancestors(ref.random_parents(rng, n)) if n else [])]
        if not tree:
            paths = [list(range(i + 1)) for n in sizes for i in range(n)]
        words = (max(sizes + [1]) + 31) // 32
        self.mask = ref.mask_words(paths, words) + [[-1] * words] * pad
        at = ref.indptr(sizes)
        self.paths = [[self.tokens[at[b] + j] for j in p] if path else [] for b, p in zip(self.row_of, paths)] + [[]] * pad
        f32 = lambda: torch.rand(rows, generator=g) + 0.5  # noqa: E731
        self.terms = {k: f32() if k in terms else None for k in ("repetition", "frequency", "presence")}
        self.bias = None
        if bias:
            lists = [[(ident(), rng.uniform(-9, 9)) for _ in range(rng.choice([0, bias]))] for _ in range(rows)]
            self.bias_lists = lists
            self.bias = [dict(p) for p in lists]  # (of a token listed twice the later value)
        self.allowed = (torch.rand(t, vocab, generator=g) < 0.5) if allowed else None
        if allowed and total > 1:
            self.allowed[1] = False  # nothing may follow
        self.sizes, self.tree, self.path, self.prompt = sizes, tree, path, prompt

    def args(self, dev):
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        cols = max([len(h) for h in self.history] + [0]) + 2
        # What lies behind a history's end must not count.
        hist = [h + [0] * (cols - len(h)) for h in self.history]
        kw = dict(history=i32(hist), history_len=i32([len(h) for h in self.history]), indptr=i32(ref.indptr(self.sizes)))
        if self.prompt:
            kw["prompt_len"] = i32(self.prompts)
        if self.path:
            kw["tokens"] = i32(self.tokens)
            if self.tree:
                kw["tree_mask"] = i32(self.mask)
        kw.update({k: v.to(dev) for k, v in self.terms.items() if v is not None})
        if self.bias is not None:
            flat = [p for r in self.bias_lists for p in r]
            kw["bias"] = (i32(ref.indptr([len(r) for r in self.bias_lists])), i32([a for a, _ in flat]),
                          torch.tensor([w for _, w in flat], dtype=torch.float32, device=dev))
        if self.allowed is not None:
            kw["allowed"] = _pack(self.allowed).to(dev)
        return kw

    def check(self, dev):
        x32, x64, bound = ref.adjust(self.logits, self.row_of, self.history, self.prompts, self.paths, *(
            self.terms[k] for k in ("repetition", "frequency", "presence")), self.bias, self.allowed)
        base = self.base.to(dev)
        logits = base[:, :self.logits.shape[1]]
        kw = self.args(dev)
        got = adjust_logits(logits, **kw)
        ids = pick_tokens(logits, **kw)
        assert torch.equal(base.cpu(), self.base), "the logits were changed"
        # The fp32 steps and their one rounding, and the definition with its bound.
        assert torch.equal(got.cpu(), x32.to(self.logits.dtype))
        d = (got.double().cpu() - x64).abs()
        fin = torch.isfinite(x64)
        assert bool((d[fin] <= bound[fin]).all())
        assert bool((got.double().cpu()[~fin] == x64[~fin]).all())
        assert ids.cpu().tolist() == ref.pick(x32, self.row_of)
        # In place, the columns behind the vocabulary untouched.
        assert adjust_logits(logits, out=logits, **kw) is logits
        assert torch.equal(logits, got)
        assert torch.equal(base[:, self.logits.shape[1]:].cpu(), self.base[:, self.logits.shape[1]:])


DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,vocab", [([1], 1), ([1], 31), ([3, 0, 2], 1000), ([1, 1, 1], 32001), ([40, 7], 517),
                                         ([2, 5], 60000)])
def test_everything_at_once(cuda_device, sizes, vocab, dtype):
    Case(vocab, sizes, vocab, dtype, bias=9, allowed=True, pad=2).check(cuda_device)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("row_pad", [1, 3, 8])
def test_rows_at_any_alignment(cuda_device, dtype, row_pad):
    Case(row_pad, [2, 3], 4099, dtype, bias=5, allowed=True, row_pad=row_pad).check(cuda_device)


@pytest.mark.parametrize("terms", [(), ("repetition",), ("frequency",), ("presence",)])
def test_terms_alone(cuda_device, terms):
    Case(len(terms), [4, 1, 9], 777, torch.bfloat16, terms=terms).check(cuda_device)


@pytest.mark.parametrize("kw", [dict(tree=False), dict(path=False), dict(prompt=False), dict(hist=0),
                                dict(hist=5000, dense=True), dict(bias=300, dense=True), dict(hist=3000, bias=40)])
def test_what_counts(cuda_device, kw):
    Case(3, [5, 2, 0, 33], 2500, torch.float32, **kw).check(cuda_device)


def test_one_row_a_token_without_indptr(cuda_device):
    c = Case(5, [1] * 6, 3001, torch.bfloat16)
    kw = c.args(cuda_device)
    x = c.logits.to(cuda_device)
    want = pick_tokens(x, **kw)
    kw.pop("indptr")
    assert torch.equal(pick_tokens(x, **kw), want)


def test_nothing_but_logits(cuda_device):
    x = torch.randn(3, 5000, device=cuda_device).to(torch.bfloat16)
    assert torch.equal(adjust_logits(x), x)
    assert torch.equal(pick_tokens(x).long(), torch.tensor(ref.pick(x.float().cpu(), [0] * 3), device=cuda_device))


def test_ties_nan_and_infinities(cuda_device):
    x = torch.zeros(6, 70000, device=cuda_device)
    x[0, [5, 6, 69999]] = 3.0
    x[1, 1000] = math.nan
    x[1, 60000] = 2.0
    x[2] = -math.inf
    x[3] = math.nan
    x[4, 40000] = math.inf
    x[4, 50000] = math.inf
    x[5] = -math.inf
    x[5, 69999] = -1e38
    want = [5, 60000, -1, -1, 40000, 69999]
    for dtype in (torch.float32, torch.bfloat16):
        assert pick_tokens(x.to(dtype)).tolist() == want
    # NaN and infinities in places that are not allowed are -inf.
    allowed = torch.zeros(6, 70000, dtype=torch.bool)
    allowed[:, 7:90] = True
    words = _pack(allowed).to(cuda_device)
    assert pick_tokens(x, allowed=words).tolist() == [7, 7, -1, -1, 7, -1]
    y = adjust_logits(x, allowed=words)
    assert bool((y.cpu()[~allowed] == -math.inf).all())


def test_ids_outside_the_vocabulary_do_not_count(cuda_device):
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda_device)  # noqa: E731
    x = torch.randn(1, 300, device=cuda_device)
    y = adjust_logits(x, history=i32([[-1, 300, 2 ** 31 - 1, -2 ** 31]]), history_len=i32([4]), tokens=i32([400]),
                      frequency=torch.ones(1, device=cuda_device),
                      bias=(i32([0, 2]), i32([-3, 300]), torch.ones(2, device=cuda_device)))
    assert torch.equal(x, y)


def test_lengths_and_prefix_sums_out_of_range(cuda_device):
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda_device)  # noqa: E731
    x = torch.zeros(2, 300, device=cuda_device)
    one = torch.ones(2, device=cuda_device)
    status = i32([0])
    y = adjust_logits(x, history=i32([[4, 5], [6, 7]]), history_len=i32([99, -3]), frequency=one)
    assert y[0, [4, 5]].tolist() == [-1.0, -1.0] and bool((y[1] == 0).all())
    adjust_logits(x, indptr=i32([0, 5, 2]), frequency=one, status=status)
    assert int(status) == 4
    status.zero_()
    adjust_logits(x, bias=(i32([0, 9, 9]), i32([1, 2]), one), status=status)
    assert int(status) == 4


@pytest.mark.parametrize("vocab", [1000, 40003])
def test_rows_that_overlap(cuda_device, vocab):
    """Prefix sums that go back: rows whose lists share memory stay within their logits, and the status says so."""
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda_device)  # noqa: E731
    x = torch.randn(40, vocab, generator=torch.Generator().manual_seed(1)).to(cuda_device)
    tokens = i32([(7919 * i) % vocab for i in range(40)])
    status = i32([0])
    kw = dict(indptr=i32([0, 30, 2, 40, 1, 40]), tokens=tokens, frequency=torch.ones(5, device=cuda_device), status=status)
    for _ in range(3):
        out = adjust_logits(x, **kw)
        ids = pick_tokens(x, **kw)
        assert int(status) == 4
        changed = (out != x).nonzero()
        assert set(changed[:, 1].tolist()) <= set(tokens.tolist())
        assert bool(((ids >= -1) & (ids < vocab)).all())


def test_replayed_with_other_histories(cuda_device):
    c = Case(8, [3, 4], 9001, torch.bfloat16, bias=7, allowed=True)
    kw = c.args(cuda_device)
    x = c.logits.to(cuda_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pick_tokens(x, **kw)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ids, out = pick_tokens(x, **kw), adjust_logits(x, **kw)
    for n in (1, 0, 30):
        kw["history_len"].fill_(n)
        kw["history"].random_(0, 9001)
        g.replay()
        assert torch.equal(ids, pick_tokens(x, **kw)) and torch.equal(out, adjust_logits(x, **kw))


def test_histories_past_16_bits(cuda_device):
    """70000 tokens, some of them more than 65535 times."""
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda_device)  # noqa: E731
    n = 70000
    history = torch.full((2, n), 7, dtype=torch.int32, device=cuda_device)
    history[0, 66000:] = 2999
    history[1, :100] = 5
    x = torch.zeros(2, 3000, device=cuda_device)
    y = adjust_logits(x, history=history, history_len=i32([n, n]), prompt_len=i32([10, 50]),
                      frequency=torch.ones(2, device=cuda_device))
    want = torch.zeros(2, 3000)
    want[0, 7], want[0, 2999], want[1, 5], want[1, 7] = -65990, -4000, -50, -69900
    assert torch.equal(y.cpu(), want)


@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 140001), (torch.bfloat16, 270000)])
def test_many_tokens_of_large_vocabularies(cuda_device, dtype, vocab):
    """More chunks a warp than it looks up at once, against the same rows in small calls."""
    g = torch.Generator(device=cuda_device).manual_seed(1)
    rows = 460
    x = (torch.randn(rows, vocab, generator=g, device=cuda_device) * 3).to(dtype)
    history = (torch.rand(rows, 3000, generator=g, device=cuda_device).pow(2) * vocab).int()
    length = torch.full((rows,), 3000, dtype=torch.int32, device=cuda_device)
    terms = {k: torch.rand(rows, generator=g, device=cuda_device) + 0.5 for k in ("repetition", "frequency", "presence")}
    whole, ids = (f(x, history=history, history_len=length, **terms) for f in (adjust_logits, pick_tokens))
    for a in range(0, rows, 46):
        part = slice(a, a + 46)
        kw = dict(history=history[part], history_len=length[part], **{k: v[part] for k, v in terms.items()})
        assert torch.equal(adjust_logits(x[part], **kw), whole[part])
        assert torch.equal(pick_tokens(x[part], **kw), ids[part])
    # (Of equal values the lowest id: the rounded logits cannot tell which the larger one was.)
    top = whole.float().max(1).values
    assert bool((whole.float().gather(1, ids.long()[:, None])[:, 0] == top).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,vocab", [([3, 0, 2], 1000), ([40, 7, 1], 9001), ([2, 5], 60000)])
def test_long_buffers_of_short_histories(cuda_device, sizes, vocab, dtype):
    """The marks' lists lie by the vocabulary's parts where those are less than the rows' buffers."""
    c = Case(vocab + 1, sizes, vocab, dtype, hist=200, bias=30, allowed=True, pad=1)
    kw, x = c.args(cuda_device), c.logits.to(cuda_device)
    want = adjust_logits(x, **kw), pick_tokens(x, **kw)
    for cols in (5000, 70000):
        longer = torch.randint(0, vocab, (len(sizes), cols), dtype=torch.int32, device=cuda_device)
        longer[:, :kw["history"].shape[1]] = kw["history"]
        for b, h in enumerate(c.history):
            longer[b, :len(h)] = torch.tensor(h, dtype=torch.int32, device=cuda_device)
        kw["history"] = longer
        assert torch.equal(adjust_logits(x, **kw), want[0]) and torch.equal(pick_tokens(x, **kw), want[1])


def test_lists_are_bounded_by_the_vocabulary(cuda_device):
    """4096 rows of 2^19 history columns: 2^31 places, of which 4096 rows of 5000 entries can be touched."""
    rows, cols, vocab = 4096, 2 ** 19, 5000
    g = torch.Generator(device=cuda_device).manual_seed(2)
    one = torch.randint(0, vocab, (1, cols), generator=g, device=cuda_device, dtype=torch.int32)
    length = torch.tensor([0, 1, 17, 1000], device=cuda_device, dtype=torch.int32).repeat(rows // 4)
    length[0] = cols
    y = adjust_logits(torch.zeros(rows, vocab, device=cuda_device), history=one.expand(rows, cols), history_len=length,
                      frequency=torch.ones(rows, device=cuda_device))
    for b in (0, 1, 2, 3, rows - 2, rows - 1):
        counts = torch.bincount(one[0, :int(length[b])].long(), minlength=vocab)
        assert torch.equal(y[b], -counts.float())
    assert torch.equal(y[4:8].repeat(rows // 4 - 1, 1), y[4:])
    # The workspace of 64 rows: what 151936 entries a row can fill, not what 131072 columns a marking CTA could.
    a = _capi.AspireLogitsArgs()
    a.logits, a.type, a.tokens, a.rows, a.vocab, a.logits_stride, a.out, a.out_stride = 256, 0, 64, 64, 151936, 151936, 256, 151936
    a.history, a.history_len, a.history_cols, a.history_stride, a.frequency = 256, 256, 131072, 131072, 256
    assert 64 * 151936 * 8 <= _capi.load_library().aspire_logits_workspace(a) <= 1.1 * 64 * 151936 * 8


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("negative", [False, True])
def test_nan_and_infinities_under_penalties(cuda_device, dtype, negative):
    """On listed entries too; with terms below their neutral values an infinity may turn."""
    c = Case(31, [3, 9, 1], 3001, dtype, hist=400, bias=20, allowed=True)
    g = torch.Generator().manual_seed(31)
    kind = torch.rand(c.base.shape, generator=g)
    for value, lo in ((math.nan, 0.0), (math.inf, 0.02), (-math.inf, 0.04)):
        c.base[(kind >= lo) & (kind < lo + 0.02)] = value
    c.base[3] = -math.inf  # nothing but listed entries could rise
    c.base[4] = math.nan
    if negative:
        c.terms = {k: -v for k, v in c.terms.items()}
    for b, lists in enumerate(c.bias_lists):
        if lists:
            lists[0] = (lists[0][0], math.inf)
            c.bias[b] = dict(lists)
    x32, _, _ = ref.adjust(c.logits, c.row_of, c.history, c.prompts, c.paths, *(
        c.terms[k] for k in ("repetition", "frequency", "presence")), c.bias, c.allowed)
    x, kw = c.logits.to(cuda_device), c.args(cuda_device)
    got, want = adjust_logits(x, **kw).cpu(), x32.to(dtype)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.5), want.nan_to_num(0.5))
    assert pick_tokens(x, **kw).tolist() == ref.pick(x32, c.row_of)
