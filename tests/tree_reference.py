"""Definitions of a tree-speculation step's operators for their tests, in
Python integers and 64-bit floats on the CPU, and the error bounds that follow
from how the kernels round.
"""

from __future__ import annotations

import math
import random

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def random_parents(rng: random.Random, nodes: int, reach: int = 6) -> list[int]:
    return [-1] + [rng.randint(max(0, i - reach), i - 1) for i in range(1, nodes)]


def ancestors(parents: list[int]) -> list[list[int]]:
    """Every node's path from the root, itself included."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if p >= 0 else []) + [i])
    return out


def mask_words(paths: list[list[int]], words: int) -> list[list[int]]:
    rows = []
    for path in paths:
        row = [0] * words
        for j in path:
            if j < 32 * words:
                row[j // 32] |= 1 << (j % 32)
        rows.append([v - (1 << 32) if v >= 1 << 31 else v for v in row])
    return rows


def indptr(counts) -> list[int]:
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


# ------------------------------------------------------------- step tables
def step_tables(lengths, new, table, held, free, count, page, tokens, parents=None, words=0):
    """Dicts of lists; `table`, `held` and `free` change in place, the new count comes back."""
    rows = len(lengths)
    cols = len(table[0]) if rows else 0
    bad = 0
    want, fits = [], []
    for b in range(rows):
        w = -(-(lengths[b] + new[b]) // page)
        ok = w <= cols and (parents is None or new[b] <= 32 * words)
        fits.append(ok)
        want.append(w if ok else held[b])
        bad |= 0 if ok else 4
    for b in range(rows):
        for c in range(want[b], held[b]):
            free[count] = table[b][c]
            table[b][c] = -1
            count += 1
    served, used = [], 0
    for b in range(rows):
        need = max(0, want[b] - held[b])
        ok = fits[b] and (need == 0 or (used + need <= count and not any(
            fits[a] and not served[a] for a in range(b))))
        served.append(ok)
        used += need if ok else 0
        bad |= 16 if fits[b] and not ok else 0
    at = count - used
    count -= used
    for b in range(rows):
        if served[b]:
            for c in range(held[b], want[b]):
                table[b][c] = free[at]
                at += 1
            held[b] = want[b]
    ends = [lengths[b] + new[b] if served[b] else 0 for b in range(rows)]
    out = {"qo_indptr": indptr(new), "kv_indptr": indptr(-(-e // page) for e in ends), "kv_len": ends,
           "last_page_len": [(e - 1) % page + 1 if e else 0 for e in ends],
           "positions": [0] * tokens, "slots": [-1] * tokens,
           "tree_mask": [[0] * words for _ in range(tokens)] if parents is not None else None}
    for b in range(rows):
        lo = out["qo_indptr"][b]
        here = None
        if parents is not None:
            here = list(parents[lo:lo + new[b]])
            for i, p in enumerate(here):
                if p >= i or p < -1:
                    here[i] = -1
                    bad |= 4
            paths = ancestors(here)
            masks = mask_words(paths, words)
        for i in range(new[b]):
            t = lo + i
            if t >= tokens:
                bad |= 4
                continue
            out["positions"][t] = lengths[b] + (len(paths[i]) - 1 if here is not None else i)
            if here is not None:
                out["tree_mask"][t] = masks[i]
            place = lengths[b] + i
            if served[b]:
                out["slots"][t] = table[b][place // page] * page + place % page
    return out, count, bad


# --------------------------------------------------------------- attention
def tree_attention(q, cache, pages, starts, ends, seen):
    """(out, lse base 2, bound of out, bound of lse) in 64 bits.

    `pages[b]` lists row b's pages, `starts` its first query row (and one past
    the last row's), `ends` its keys, `seen[b]` bool [queries, queries].

    Bounds: the products of bf16 are exact in fp32 and each of the 128
    additions loses at most 2^-22 of the sum of magnitudes (the matrix
    instructions may truncate); the exponent's argument and ex2 lose 2^-21 of
    1 + |x|; P is rounded to bf16 (2^-8) before the second product, whose sum
    over n keys loses n 2^-22; the joined chunks 2^-20; the output is rounded
    to bf16."""
    heads, kv = q.shape[1], cache.shape[3]
    scale = 128 ** -0.5
    out = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    bound = torch.zeros_like(out)
    lbound = torch.zeros_like(lse)
    for b, end in enumerate(ends):
        lo, n = starts[b], starts[b + 1] - starts[b]
        if end == 0 or n == 0:
            continue
        both = cache[torch.tensor(pages[b])].double().permute(1, 3, 0, 2, 4).reshape(2, kv, -1, 128)[:, :, :end]
        sees = torch.zeros(n, end, dtype=torch.bool)
        sees[:, :max(0, end - n)] = True
        first = max(0, n - end)  # nodes whose keys lie before the cache's first place
        sees[:, max(0, end - n):] = seen[b][:, first:]
        for h in range(heads):
            k, v = both[0, h * kv // heads], both[1, h * kv // heads]
            qh = q[lo:lo + n, h].double()
            x = (qh @ k.t()) * scale
            err = (qh.abs() @ k.abs().t()) * scale * 128 * 2.0 ** -22 + (1 + x.abs()) * 2.0 ** -21
            x = x.masked_fill(~sees, -math.inf)
            some = sees.any(1)
            l = torch.logsumexp(x, 1)
            p = torch.where(some[:, None], torch.exp(x - torch.where(some, l, 0.0)[:, None]), 0.0)
            rel = torch.where(sees, err, 0.0)
            worst = rel.amax(1, keepdim=True)
            o = p @ v
            out[lo:lo + n, h] = o
            lse[lo:lo + n, h] = torch.where(some, l / math.log(2.0), -math.inf)
            mag = p @ v.abs()
            bound[lo:lo + n, h] = mag * (2.0 ** -8 + 2 * worst + end * 2.0 ** -22 + 2.0 ** -20) * 1.01 + o.abs() * 2.0 ** -8
            lbound[lo:lo + n, h] = (worst[:, 0] + 2.0 ** -19) * 1.5 + torch.where(some, l.abs(), 0.0) * 2.0 ** -20
    return out, lse, bound, lbound


# ------------------------------------------------------------------ logits
def adjust(logits, rows, history, prompts, paths, repetition, frequency, presence, bias, allowed):
    """(value, exact value in 64 bits, bound) [tokens, vocab] of token t of row
    rows[t] (-1: none): fp32 step by step, and the definition.  `history[b]`
    lists ids, its first prompts[b] the prompt; `paths[t]` the path's ids;
    `bias[b]` a dict; `allowed` bool [tokens, vocab] or None."""
    vocab = logits.shape[1]
    x32 = logits.float().clone()
    x64 = logits.double().clone()
    err = torch.zeros_like(x64)
    u = 2.0 ** -24
    for t, b in enumerate(rows):
        if b < 0:
            continue
        made, known = {}, set()
        for i, v in enumerate(history[b]):
            known.add(v)
            if i >= prompts[b]:
                made[v] = made.get(v, 0) + 1
        for v in paths[t]:
            known.add(v)
            made[v] = made.get(v, 0) + 1
        for v in known | set(bias[b] if bias else {}):
            if not 0 <= v < vocab:
                continue
            a, d, e = x32[t, v].clone(), x64[t, v].clone(), 0.0
            if v in known and repetition is not None:
                r = repetition[b]
                a = a / r if a > 0 else a * r
                d = d / r.double() if d > 0 else d * r.double()
                e = float(d.abs()) * u
            c = made.get(v, 0)
            if c and frequency is not None:
                a = a - frequency[b] * torch.tensor(float(c))
                d = d - frequency[b].double() * c
                e += (float(frequency[b].abs()) * c + float(d.abs())) * 2 * u
            if c and presence is not None:
                a = a - presence[b]
                d = d - presence[b].double()
                e += float(d.abs()) * 2 * u
            if bias and v in bias[b]:
                w = torch.tensor(bias[b][v], dtype=torch.float32)
                a = a + w
                d = d + w.double()
                e += float(d.abs()) * 2 * u
            x32[t, v], x64[t, v], err[t, v] = a, d, e
        if allowed is not None:
            x32[t, ~allowed[t]] = -math.inf
            x64[t, ~allowed[t]] = -math.inf
    bound = torch.where(torch.isfinite(x64), err + x64.abs() * U[logits.dtype], 0.0)
    if logits.dtype == torch.float16:
        bound = bound + 2.0 ** -25
    return x32, x64, bound


def pick(x32, rows):
    """The largest value's lowest id; NaN and -inf never; -1 for none."""
    out = []
    for t, b in enumerate(rows):
        x = torch.where(torch.isnan(x32[t]), -math.inf, x32[t])
        big = x.max()
        out.append(int((x == big).nonzero()[0, 0]) if b >= 0 and big > -math.inf else -1)
    return out


# ------------------------------------------------------------------ accept
def walk(tokens, parents, targets, most):
    """The accepted path of one row."""
    if not tokens:
        return []
    path = [0]
    while len(path) < most:
        node = path[-1]
        kids = [c for c in range(node + 1, len(tokens)) if parents[c] == node and tokens[c] == targets[node]]
        if not kids:
            break
        path.append(kids[0])
    return path
