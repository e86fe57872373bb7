"""Cases, plain forms and 64-bit definitions of the operators of tree speculation.

A row (request) holds ``length`` committed tokens in a paged cache and brings
``new`` tokens to a step: node 0 is its last committed token, which is not in
the cache yet, the others are drafts, each the child of an earlier node.

``tables``  block tables and slot maps from the rows' lengths: pages taken from
            and given back to a stack of free pages, prefix sums, positions,
            cache slots and the nodes' ancestor masks; a pass reserves for the
            new tokens and then trims to the committed ones, as a step does
            before and after its forward, so the state comes back to where it was.
``tree``    attention of the nodes over the cache: all of the committed tokens
            and the node's ancestors (mask bits).
``logits``  penalties for repeated tokens (history and path), biases and
            grammar masks on the target's logits, or the best token of those.
``accept``  the walk along the target's choices and the move of the walked
            nodes' keys and values to their committed places, all layers.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
PAGE = 16
DIM = 128


# ------------------------------------------------------------------- cases
def listed():
    return [
        # One row with a short chain of drafts: the launch's latency.
        {"name": "tables_row_1", "op": "tables", "rows": 1, "nodes": 5, "context": 700, "tree": False},
        # A decode step of 64 rows with trees of up to 48 nodes.
        {"name": "tables_trees_64", "op": "tables", "rows": 64, "nodes": 48, "context": 32768, "tree": True},
        # Prefill chunks of a full batch: many tokens a row, many new pages.
        {"name": "tables_prefill_256", "op": "tables", "rows": 256, "nodes": 2048, "context": 8192, "tree": False},
        # One row with a small tree right after a short prompt, 8 KV heads.
        {"name": "tree_short_1", "op": "tree", "rows": 1, "nodes": 5, "context": 130, "heads": 16, "kv_heads": 8},
        # A decode step of 16 rows of ragged contexts, 16 nodes each at most.
        {"name": "tree_batch_16", "op": "tree", "rows": 16, "nodes": 16, "context": 8192, "heads": 32, "kv_heads": 8},
        # Wide trees: more packed query rows than one decode tile holds.
        {"name": "tree_wide_8", "op": "tree", "rows": 8, "nodes": 64, "context": 16384, "heads": 32, "kv_heads": 8},
        # Two rows of a long context, odd sizes.
        {"name": "tree_long_2", "op": "tree", "rows": 2, "nodes": 11, "context": 131001, "heads": 32, "kv_heads": 8},
        # The next token of one row under penalties and a grammar.
        {"name": "pick_row_1", "op": "logits", "rows": 1, "nodes": 1, "history": 900, "vocab": 151936, "dtype": "bf16",
         "bias": 0, "allowed": True, "pick": True},
        # A decode step of 64 rows with long histories, biases, fp32 logits.
        {"name": "adjust_batch_64", "op": "logits", "rows": 64, "nodes": 1, "history": 16384, "vocab": 151936,
         "dtype": "f32", "bias": 64, "allowed": False, "pick": False},
        # The nodes of 16 rows' trees under penalties and grammars.
        {"name": "pick_trees_16", "op": "logits", "rows": 16, "nodes": 24, "history": 4001, "vocab": 128256,
         "dtype": "bf16", "bias": 0, "allowed": True, "pick": True},
        # One row's tree accepted in a 28-layer cache.
        {"name": "accept_row_1", "op": "accept", "rows": 1, "nodes": 9, "path": 5, "layers": 28, "kv_heads": 8},
        # A batch of trees in a 36-layer cache.
        {"name": "accept_batch_64", "op": "accept", "rows": 64, "nodes": 33, "path": 7, "layers": 36, "kv_heads": 8},
    ]


def draw(rng):
    def spread(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    most = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    while True:
        op = rng.choice(["tables", "tree", "tree", "logits", "logits", "accept"])
        if op == "tables":
            tree = rng.random() < 0.5
            case = {"op": op, "rows": spread(1, 256), "nodes": spread(1, 64 if tree else 2048),
                    "context": spread(16, 32768), "tree": tree}
        elif op == "tree":
            kv_heads = rng.choice([1, 2, 4, 8])
            case = {"op": op, "rows": spread(1, 48), "nodes": spread(1, 80), "context": spread(16, 65536),
                    "heads": kv_heads * rng.choice([1, 2, 4, 5, 8]), "kv_heads": kv_heads}
        elif op == "logits":
            case = {"op": op, "rows": spread(1, 96), "nodes": rng.choice([1, 1, spread(2, 32)]),
                    "history": spread(1, 32768), "vocab": rng.choice([32000, 50001, 128256, 151936]),
                    "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "bias": rng.choice([0, spread(1, 256)]),
                    "allowed": rng.random() < 0.5, "pick": rng.random() < 0.5}
        else:
            case = {"op": op, "rows": spread(1, 96), "nodes": spread(2, 64), "path": spread(2, 12),
                    "layers": rng.choice([12, 28, 32, 36]), "kv_heads": rng.choice([1, 2, 4, 8])}
        w = work(case)
        if all(w[k] <= most[k] for k in most):
            return case


def _sizes(case):
    """Committed lengths (or histories) and nodes of the rows: ragged, the first row the longest."""
    rng = random.Random(case["rows"] * 1000003 + case["nodes"])
    n, most = case["rows"], case.get("context", case.get("history"))
    lengths = [most] + [rng.randint(most // 4, most) for _ in range(n - 1)]
    nodes = [case["nodes"]] + [rng.randint(max(1, case["nodes"] // 2), case["nodes"]) for _ in range(n - 1)]
    return lengths, nodes


def _walk(case, row):
    """Nodes after node 0 on a row's accepted path, and whether they already lie in their places (a first branch)."""
    n = case["nodes"] if row == 0 else max(1, case["nodes"] - row % 5)
    m = min(1 + row % max(1, case["path"] - 1), n - 1)
    return n, m, row % 3 == 2 or n - 1 - m < m


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _indptr(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def _parents(rng, nodes):
    """A row's tree: a node hangs on one of the eight before it."""
    return [-1] + [rng.randint(max(0, i - 8), i - 1) for i in range(1, nodes)]


def _mask_words(parents, words):
    """Ancestor bits (self included) of a row's nodes, 32 to a word."""
    bits = []
    for i, p in enumerate(parents):
        bits.append((1 << i) | (bits[p] if p >= 0 else 0))
    out = []
    for b in bits:
        for w in range(words):
            v = (b >> (32 * w)) & 0xFFFFFFFF
            out.append(v - (1 << 32) if v >= 1 << 31 else v)
    return out


def _prepare_tables(case, seed):
    g = _gen(seed)
    rng = random.Random(seed)
    b, n = case["rows"], case["nodes"]
    lengths = [rng.randint(case["context"] // 4, case["context"]) for _ in range(b)]
    # Every sixteenth row is idle or finished.
    new = [0 if i % 16 == 15 else rng.randint(max(1, n // 2), n) for i in range(b)]
    held = [(v + PAGE - 1) // PAGE for v in lengths]
    cols = (case["context"] + n + PAGE - 1) // PAGE + 1
    spare = b * cols - sum(held)
    ids = torch.randperm(b * cols, generator=g, device="cuda").to(torch.int32)
    table = torch.full((b, cols), -1, dtype=torch.int32, device="cuda")
    held_t = _i32(held)
    table[torch.arange(cols, device="cuda")[None, :] < held_t[:, None]] = ids[:sum(held)]
    # The stack of free pages has room for every page.
    free = torch.zeros(ids.numel(), dtype=torch.int32, device="cuda")
    free[:spare] = ids[sum(held):]
    s = {"case": case, "lengths": _i32(lengths), "new": _i32(new), "idle": torch.zeros(b, dtype=torch.int32, device="cuda"),
         "table": table, "held": held_t, "free": free, "count": _i32([spare]), "tokens": b * n, "parents": None}
    if case["tree"]:
        p = [v for c in new for v in (_parents(rng, c) if c else [])]
        s["parents"] = _i32(p + [0] * (b * n - len(p)))
    return s


def _prepare_tree(case, seed):
    g = _gen(seed)
    rng = random.Random(seed)
    lengths, nodes = _sizes(case)
    ends = [a + c for a, c in zip(lengths, nodes)]
    pages = [(v + PAGE - 1) // PAGE for v in ends]
    cols = max(pages)
    ids = torch.randperm(sum(pages), generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(case["rows"], cols, dtype=torch.int32, device="cuda")
    table[torch.arange(cols, device="cuda")[None, :] < _i32(pages)[:, None]] = ids
    words = (max(nodes) + 31) // 32
    mask = [w for c in nodes for w in _mask_words(_parents(rng, c), words)]
    cache = torch.empty(sum(pages), 2, PAGE, case["kv_heads"], DIM, dtype=torch.bfloat16, device="cuda")
    cache.normal_(generator=g)
    q = torch.empty(sum(nodes), case["heads"], DIM, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    s = {"case": case, "q": q, "cache": cache, "table": table, "mask": _i32(mask).view(-1, words),
         "modes": torch.ones(case["rows"], dtype=torch.int32, device="cuda"), "qo": _indptr(nodes),
         "pages": _indptr(pages), "ends": ends}
    if own:
        _plan(s)
    return s


def _plan(s):
    """The attention's handle with the step's plan, which every layer of the step uses."""
    from aspire_b200.attention import HolisticAttentionWrapper

    case = s["case"]
    w = HolisticAttentionWrapper(s["q"])
    w.set_page_tables(s["modes"], s["table"], s["table"])
    w.plan_host(torch.tensor(s["qo"]), torch.tensor(s["pages"]), torch.tensor(s["ends"]), None, case["heads"],
                case["kv_heads"], DIM, PAGE, causal=False)
    s["handle"] = w


def _prepare_logits(case, seed):
    g = _gen(seed)
    rng = random.Random(seed)
    b, v = case["rows"], case["vocab"]
    lens, nodes = _sizes(case)
    t = b * case["nodes"]  # the step's buffers; rows past the last node are padding
    rand = lambda *shape: torch.rand(*shape, generator=g, device="cuda")  # noqa: E731
    # Few tokens make most of a text.
    history = (rand(b, case["history"] + 3).pow(3) * v).to(torch.int32).clamp_(max=v - 1)
    words = (max(nodes) + 31) // 32
    mask = [w for c in nodes for w in _mask_words(_parents(rng, c), words)]
    logits = torch.empty(t, v, device="cuda").normal_(generator=g).mul_(3).to(DTYPES[case["dtype"]])
    s = {"case": case, "logits": logits, "history": history, "history_len": _i32(lens),
         "prompt_len": _i32([c // 2 for c in lens]), "repetition": 1 + 0.3 * rand(b), "frequency": 0.5 * rand(b),
         "presence": 0.5 * rand(b), "indptr": _i32(_indptr(nodes)),
         "tokens": (rand(t).pow(3) * v).to(torch.int32).clamp_(max=v - 1),
         "mask": torch.cat([_i32(mask), torch.zeros(t * words - len(mask), dtype=torch.int32, device="cuda")]).view(t, words),
         "bias": None, "allowed": None}
    if case["bias"]:
        per = [case["bias"] if i % 4 else case["bias"] // 2 for i in range(b)]
        ids = rand(b, v).topk(case["bias"], dim=1).indices.to(torch.int32)
        keep = torch.arange(case["bias"], device="cuda")[None, :] < _i32(per)[:, None]
        s["bias"] = (_i32(_indptr(per)), ids[keep], 4 * torch.randn(sum(per), generator=g, device="cuda"))
    if case["allowed"]:
        s["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (t, (v + 31) // 32), generator=g, device="cuda").to(torch.int32)
    return s


def _prepare_accept(case, seed):
    g = _gen(seed)
    rng = random.Random(seed)
    b = case["rows"]
    parents, tokens, targets, nodes, lengths = [], [], [], [], []
    for row in range(b):
        n, m, placed = _walk(case, row)
        # A branch behind the places that it moves to, so that a pass can be repeated on the same cache.
        path = list(range(1, m + 1)) if placed else sorted(rng.sample(range(m + 1, n), m))
        p = _parents(rng, n)
        for before, node in zip([0] + path, path):
            p[node] = before
        toks = rng.sample(range(100, 151936), n)
        want = [rng.randint(100, 151935) for _ in range(n)]
        for before, node in zip([0] + path, path):
            want[before] = toks[node]
        parents += p
        tokens += toks
        targets += want
        nodes.append(n)
        lengths.append(rng.randint(0, 3 * PAGE))
    ends = [a + n for a, n in zip(lengths, nodes)]
    cols = (3 * PAGE + case["nodes"] + PAGE - 1) // PAGE
    table = torch.randperm(b * cols, generator=g, device="cuda").to(torch.int32).view(b, cols)
    caches = []
    for _ in range(case["layers"]):
        c = torch.empty(b * cols, 2, PAGE, case["kv_heads"], DIM, dtype=torch.bfloat16, device="cuda")
        caches.append(c.normal_(generator=g))
    return {"case": case, "parents": _i32(parents), "tokens": _i32(tokens), "targets": _i32(targets),
            "indptr": _i32(_indptr(nodes)), "lengths": _i32(lengths), "table": table, "caches": caches, "ends": ends}


def prepare(case, seed):
    make = {"tables": _prepare_tables, "tree": _prepare_tree, "logits": _prepare_logits, "accept": _prepare_accept}
    return make[case["op"]](case, seed)


# -------------------------------------------------------------- plain form
def _plain_ancestors(parents, local, most):
    """Ancestor flags [t, most] (self included) and depth of nodes with local
    indices `local`, `parents` local too."""
    t = torch.arange(local.numel(), device=local.device)
    at, depth = local.clone(), torch.zeros_like(local)
    seen = torch.zeros(local.numel(), most + 1, dtype=torch.bool, device=local.device)
    for _ in range(most):
        seen.scatter_(1, torch.where(at >= 0, at, most)[:, None], True)
        up = parents[(t - local + at.clamp(min=0))]
        at = torch.where(at >= 0, up, -1)
        depth = depth + (at >= 0)
    return seen[:, :most], depth


def _plain_step(s, new, tokens, parents):
    """One call's tables; the block table, the pages held and the free pages change in place."""
    table, held, free, count = s["table"], s["held"], s["free"], s["count"]
    length = s["lengths"].long()
    new = new.long()
    cols = torch.arange(table.shape[1], device="cuda")[None, :]
    want = (length + new + PAGE - 1) // PAGE
    have = held.long()
    # Pages past what a row needs go on top of the stack, in row order.
    back = (cols >= want[:, None]) & (cols < have[:, None])
    at = torch.where(back, count.long() + back.flatten().cumsum(0).view(back.shape) - 1, free.numel())
    stack = torch.cat([free, free[:1]]).scatter(0, at.flatten(), table.flatten())
    avail = count.long() + back.sum()
    # Rows are served in order while there are pages; the block on top is handed out from its bottom.
    need = (want - have).clamp(min=0)
    need = torch.where(want <= table.shape[1], need, 0)
    served = (want <= table.shape[1]) & ((need == 0) | (need.cumsum(0) <= avail))
    take = (cols >= have[:, None]) & (cols < want[:, None]) & served[:, None]
    total = take.sum()
    at = torch.where(take, avail - total + take.flatten().cumsum(0).view(take.shape) - 1, 0)
    page = torch.where(take, stack[at], torch.where(back, -1, table))
    table.copy_(page)
    free.copy_(stack[:-1])
    count.copy_(avail - total)
    held.copy_(torch.where(served, want, have))
    ends = torch.where(served, length + new, 0)
    pages = (ends + PAGE - 1) // PAGE
    zero = torch.zeros(1, dtype=torch.long, device="cuda")
    qo = torch.cat([zero, new.cumsum(0)])
    out = {"qo_indptr": qo, "kv_indptr": torch.cat([zero, pages.cumsum(0)]), "kv_len": ends,
           "last_page_len": torch.where(ends > 0, (ends - 1) % PAGE + 1, 0)}
    out = {k: v.to(torch.int32) for k, v in out.items()}
    if tokens:
        t = torch.arange(tokens, device="cuda")
        live = t < qo[-1]
        row = torch.searchsorted(qo[1:], t, right=True).clamp(max=new.numel() - 1)
        local = torch.where(live, t - qo[row], 0)
        depth = local
        if parents is not None:
            most = s["case"]["nodes"]
            seen, depth = _plain_ancestors(torch.where(live, parents.long(), -1), local, most)
            words = (most + 31) // 32
            seen = torch.nn.functional.pad(seen & live[:, None], (0, 32 * words - most)).view(tokens, words, 32)
            bits = (seen.long() << torch.arange(32, device="cuda")).sum(2)
            out["tree_mask"] = torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).to(torch.int32)
        out["positions"] = torch.where(live, length[row] + depth, 0).to(torch.int32)
        place = length[row] + local
        slot = page[row, (place // PAGE).clamp(max=table.shape[1] - 1)].long() * PAGE + place % PAGE
        out["slots"] = torch.where(live & served[row], slot, -1)
    return out


def _plain_tables(s):
    grown = _plain_step(s, s["new"], s["tokens"], s["parents"])
    trimmed = _plain_step(s, s["idle"], 0, None)
    return _tables_out(s, grown, trimmed)


def _tables_out(s, grown, trimmed):
    names = ["qo_indptr", "kv_indptr", "kv_len", "last_page_len"]
    full = names + ["positions", "slots"] + (["tree_mask"] if s["parents"] is not None else [])
    out = {"grown_" + k: grown[k] for k in full}
    out.update({"trimmed_" + k: trimmed[k] for k in names})
    out.update(table=s["table"], held=s["held"], free=s["free"], count=s["count"])
    return out


def _attend(s, kind):
    """Outputs and base-2 log-sum-exps in `kind`, row by row."""
    case = s["case"]
    heads, kv = case["heads"], case["kv_heads"]
    out, lse = [], []
    for row, end in enumerate(s["ends"]):
        lo, hi = s["qo"][row], s["qo"][row + 1]
        n = hi - lo
        pages = s["table"][row, :(end + PAGE - 1) // PAGE].long()
        both = s["cache"][pages].to(kind).permute(1, 3, 0, 2, 4).reshape(2, kv, -1, DIM)[:, :, :end]
        q = s["q"][lo:hi].to(kind).view(n, kv, heads // kv, DIM).permute(1, 2, 0, 3).reshape(kv, -1, DIM)
        x = (q @ both[0].transpose(1, 2)).view(kv, heads // kv, n, end) / math.sqrt(DIM)
        j = torch.arange(n, device="cuda")
        seen = (s["mask"][lo:hi].long()[:, j // 32] >> (j % 32)) & 1
        x[..., end - n:] = torch.where(seen.bool(), x[..., end - n:], -math.inf)
        big = x.amax(-1, keepdim=True)
        p = torch.exp(x - big)
        total = p.sum(-1, keepdim=True)
        o = ((p / total).view(kv, -1, end) @ both[1]).view(kv, heads // kv, n, DIM)
        out.append(o.permute(2, 0, 1, 3).reshape(n, heads, DIM))
        lse.append(((big + torch.log(total)) / math.log(2.0))[..., 0].permute(2, 0, 1).reshape(n, heads))
    return torch.cat(out), torch.cat(lse)


def _plain_tree(s):
    out, lse = _attend(s, torch.float32)
    return out.to(torch.bfloat16), lse


def _counts(s, token_row, live):
    """Occurrences among the outputs (history and path) and in the prompt, [t, vocab]."""
    case = s["case"]
    b, v = case["rows"], case["vocab"]
    at = torch.arange(s["history"].shape[1], device="cuda")[None, :]
    inside = at < s["history_len"][:, None]
    prompt = at < s["prompt_len"][:, None]
    ids = s["history"].long()
    made = torch.zeros(b, v, device="cuda").scatter_add_(1, ids, (inside & ~prompt).float())
    asked = torch.zeros(b, v, device="cuda").scatter_add_(1, ids, (inside & prompt).float()) > 0
    made, asked = made[token_row], asked[token_row]
    first = s["indptr"].long()[token_row]
    j = torch.arange(case["nodes"], device="cuda")
    seen = (s["mask"].long()[:, j // 32] >> (j % 32)) & 1
    path = s["tokens"].long()[(first[:, None] + j).clamp(max=s["tokens"].numel() - 1)]
    made.scatter_add_(1, path, (seen * live[:, None]).float())
    return made, asked


def _plain_logits(s):
    case = s["case"]
    t, v = s["logits"].shape
    n = torch.arange(t, device="cuda")
    ends = s["indptr"].long()
    live = n < ends[-1]
    row = torch.searchsorted(ends[1:], n, right=True).clamp(max=case["rows"] - 1)
    made, asked = _counts(s, row, live)
    x = s["logits"].float()
    r = s["repetition"][row][:, None]
    y = torch.where((made > 0) | asked, torch.where(x > 0, x / r, x * r), x)
    y = y - s["frequency"][row][:, None] * made
    y = y - s["presence"][row][:, None] * (made > 0)
    if s["bias"] is not None:
        indptr, ids, values = s["bias"]
        owner = torch.searchsorted(indptr.long()[1:], torch.arange(ids.numel(), device="cuda"), right=True)
        extra = torch.zeros(case["rows"], v, device="cuda")
        extra[owner, ids.long()] = values
        y = y + extra[row]
    if s["allowed"] is not None:
        bit = torch.arange(32, device="cuda", dtype=torch.int32)
        ok = ((s["allowed"][:, :, None] >> bit) & 1).view(t, -1)[:, :v]
        y = torch.where(ok != 0, y, -math.inf)
    if case["pick"]:
        y = torch.where(y != y, -math.inf, y)
        big = y.amax(1, keepdim=True)
        best = torch.where(y == big, torch.arange(v, device="cuda"), v).amin(1)
        return torch.where(live & (big[:, 0] > -math.inf), best, -1).to(torch.int32)
    return torch.where(live[:, None], y, x).to(s["logits"].dtype)


def _plain_accept(s):
    case = s["case"]
    b, most = case["rows"], case["path"]
    t = s["tokens"].numel()
    n = torch.arange(t, device="cuda")
    ends = s["indptr"].long()
    row = torch.searchsorted(ends[1:], n, right=True)
    local = n - ends[row]
    node = torch.zeros(b, dtype=torch.long, device="cuda")
    alive = ends[1:] > ends[:-1]
    path = torch.full((b, most), -1, dtype=torch.long, device="cuda")
    for d in range(most):
        path[:, d] = torch.where(alive, node, -1)
        want = s["targets"].long()[(ends[:-1] + node).clamp(max=t - 1)]
        hit = (s["parents"] == node[row]) & (s["tokens"] == want[row]) & alive[row]
        child = torch.full((b,), t, dtype=torch.long, device="cuda")
        child = child.scatter_reduce(0, row, torch.where(hit, local, t), "amin")
        alive = child < t
        node = torch.where(alive, child, 0)
    on = path >= 0
    count = on.sum(1)
    got = torch.where(on, s["targets"][(ends[:-1, None] + path.clamp(min=0)).clamp(max=t - 1)].long(), -1)
    to = torch.arange(most, device="cuda")[None, :]
    table = s["table"]
    place = lambda i: (table.gather(1, ((s["lengths"].long()[:, None] + i) // PAGE).clamp(max=table.shape[1] - 1)).long(),  # noqa: E731
                       (s["lengths"].long()[:, None] + i) % PAGE)
    (sp, so), (dp, do) = place(path.clamp(min=0)), place(to.expand(b, -1))
    for c in s["caches"]:
        c[dp, :, do] = torch.where(on[:, :, None, None, None], c[sp, :, so], c[dp, :, do])
    return _accept_out(s, count, path, got, s["lengths"] + count)


def _accept_out(s, count, path, tokens, lengths):
    out = {"count": count.to(torch.int32), "path": path.to(torch.int32), "tokens": tokens.to(torch.int32),
           "lengths": lengths.to(torch.int32)}
    out.update({f"cache{i}": c for i, c in enumerate(s["caches"])})
    return out


def _plain(s):
    forms = {"tables": _plain_tables, "tree": _plain_tree, "logits": _plain_logits, "accept": _plain_accept}
    with torch.no_grad():
        return forms[s["case"]["op"]](s)


# ------------------------------------------------------------- the calls
def _own(s):
    case = s["case"]
    if case["op"] == "tables":
        from aspire_b200.kv_ops import build_step_tables

        pool = (s["table"], s["held"], s["free"], s["count"])
        grown = build_step_tables(s["lengths"], s["new"], *pool, tokens=s["tokens"], parents=s["parents"],
                                  max_nodes=case["nodes"] if case["tree"] else None)
        trimmed = build_step_tables(s["lengths"], s["idle"], *pool, tokens=0)
        return _tables_out(s, grown._asdict(), trimmed._asdict())
    if case["op"] == "tree":
        if "handle" not in s:
            _plan(s)
        return s["handle"].run(s["q"], s["cache"], tree_mask=s["mask"], return_lse=True)
    if case["op"] == "logits":
        from aspire_b200.logits import adjust_logits, pick_tokens

        call = pick_tokens if case["pick"] else adjust_logits
        return call(s["logits"], history=s["history"], history_len=s["history_len"], prompt_len=s["prompt_len"],
                    indptr=s["indptr"], tokens=s["tokens"], tree_mask=s["mask"], repetition=s["repetition"],
                    frequency=s["frequency"], presence=s["presence"], bias=s["bias"], allowed=s["allowed"])
    from aspire_b200.tree import accept_tree

    a = accept_tree(s["tokens"], s["parents"], s["targets"], s["indptr"], s["lengths"], case["path"],
                    caches=s["caches"], block_table=s["table"])
    return _accept_out(s, a.count, a.path, a.tokens, a.lengths)


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------------- work
def work(case):
    op, b = case["op"], case["rows"]
    if op == "tables":
        t = b * case["nodes"]
        words = (case["nodes"] + 31) // 32 if case["tree"] else 0
        # Per token: position and slot, with a tree its parent and mask; per row its lengths, prefix sums and new pages.
        return {"bytes": t * (12 + (4 + 4 * words if case["tree"] else 0)) + b * (64 + case["nodes"] // 4),
                "flops": 8 * t}
    if op == "tree":
        lengths, nodes = _sizes(case)
        keys = sum(lengths) + sum(nodes)
        t = sum(nodes)
        words = (max(nodes) + 31) // 32
        return {"bytes": keys * case["kv_heads"] * DIM * 4 + t * (case["heads"] * (4 * DIM + 4) + 4 * words),
                "flops": 4.0 * DIM * case["heads"] * sum(n * (a + n) for a, n in zip(lengths, nodes))}
    if op == "logits":
        lengths, nodes = _sizes(case)
        t, v = sum(nodes), case["vocab"]
        size = 4 if case["dtype"] == "f32" else 2
        bytes_ = t * v * size * (1 if case["pick"] else 2) + sum(lengths) * 4 + b * case["bias"] * 8
        bytes_ += t * v // 8 if case["allowed"] else 0
        return {"bytes": bytes_, "flops": 6 * t * v}
    moved = sum(0 if placed else m for n, m, placed in (_walk(case, r) for r in range(b)))
    return {"bytes": b * case["nodes"] * 12 + moved * case["layers"] * case["kv_heads"] * DIM * 8,
            "flops": b * case["nodes"] * case["path"]}


# ------------------------------------------------- the definition in 64 bits
def _exact_tree(s):
    """Row by row and head by head, with the softmax from its definition."""
    case = s["case"]
    group = case["heads"] // case["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    for row, end in enumerate(s["ends"]):
        lo, hi = s["qo"][row], s["qo"][row + 1]
        place = torch.arange(end, device="cuda")
        page = s["table"][row].long()[place // PAGE]
        hidden = torch.ones(hi - lo, end, dtype=torch.bool, device="cuda")
        hidden[:, :end - (hi - lo)] = False
        for j in range(hi - lo):
            hidden[:, end - (hi - lo) + j] = ((s["mask"][lo:hi, j // 32] >> (j % 32)) & 1) == 0
        for h in range(case["heads"]):
            k = s["cache"][page, 0, place % PAGE, h // group].double()
            v = s["cache"][page, 1, place % PAGE, h // group].double()
            x = (s["q"][lo:hi, h].double() @ k.t() * DIM ** -0.5).masked_fill_(hidden, -math.inf)
            lse[lo:hi, h] = torch.logsumexp(x, 1) / math.log(2.0)
            out[lo:hi, h] = torch.softmax(x, 1) @ v
    return out, lse


def _exact_logits(s):
    """Row by row: the row's outputs counted with the path's, one after the other."""
    v = s["case"]["vocab"]
    y = s["logits"].double()
    ends = s["indptr"].tolist()
    for b in range(s["case"]["rows"]):
        hist = s["history"][b, :int(s["history_len"][b])].long()
        cut = int(s["prompt_len"][b])
        made = torch.bincount(hist[cut:], minlength=v).double()
        known = torch.bincount(hist, minlength=v) > 0
        lo, hi = ends[b], ends[b + 1]
        toks = s["tokens"][lo:hi].long()
        for i in range(hi - lo):
            on = torch.tensor([(int(w) >> k) & 1 for w in s["mask"][lo + i].tolist() for k in range(32)][:hi - lo])
            path = torch.bincount(toks[on.nonzero()[:, 0].cuda()], minlength=v).double()
            c = made + path
            x = y[lo + i]
            r = s["repetition"][b].double()
            x = torch.where(known | (path > 0), torch.where(x > 0, x / r, x * r), x)
            x = x - s["frequency"][b].double() * c - s["presence"][b].double() * (c > 0)
            if s["bias"] is not None:
                at = slice(int(s["bias"][0][b]), int(s["bias"][0][b + 1]))
                x[s["bias"][1][at].long()] += s["bias"][2][at].double()
            if s["allowed"] is not None:
                word = torch.arange(v, device="cuda")
                x[(s["allowed"][lo + i][word // 32] >> (word % 32)) & 1 == 0] = -math.inf
            y[lo + i] = x
    return y


def exact(case, seed):
    if case["op"] in ("tables", "accept") or case.get("pick"):
        return None
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_tree(s) if case["op"] == "tree" else _exact_logits(s)
