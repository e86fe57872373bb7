"""The accepted path of trees of drafted tokens.

A step of tree speculation::

    t = build_step_tables(lengths, new_tokens, *pool, tokens=T, parents=parents, max_nodes=N)
    wrapper.plan_device(t.qo_indptr, t.kv_indptr, t.last_page_len, ..., trees=True)
    # per layer: qkv_prologue(..., positions=t.positions), then
    wrapper.run(q, cache, tree_mask=t.tree_mask)
    targets = pick_tokens(logits, indptr=t.qo_indptr, tokens=tokens, tree_mask=t.tree_mask, ...)
    a = accept_tree(tokens, parents, targets, t.qo_indptr, lengths, max_path, caches=caches, block_table=block_table,
                    kv_len=t.kv_len)
    build_step_tables(a.lengths, None, *pool, tokens=0)      # pages of the rejected nodes go back

Node 0 of a row is its last committed token, which is not in the cache yet;
the others are drafts.  Nothing reads a value back from the device.
"""

from __future__ import annotations

from typing import NamedTuple, Sequence

import torch

from . import _capi


class Accepted(NamedTuple):
    """``count`` int32 ``[rows]``: nodes on the accepted path, the root
    included (0 for a row without nodes, without keys in the cache, or without
    a choice after its root); ``path`` int32 ``[rows, max_path]``:
    those nodes; ``tokens`` int32 ``[rows, max_path]``: the tokens committed,
    the target's choice after each of them (the accepted drafts, then one
    more); -1 behind the path.  ``lengths`` int32 ``[rows]``: the lengths plus
    the counts."""

    count: torch.Tensor
    path: torch.Tensor
    tokens: torch.Tensor
    lengths: torch.Tensor


def accept_tree(tokens: torch.Tensor, parents: torch.Tensor, targets: torch.Tensor, indptr: torch.Tensor,
                lengths: torch.Tensor, max_path: int, *, caches: Sequence[torch.Tensor] = (),
                block_table: torch.Tensor | None = None, kv_len: torch.Tensor | None = None,
                status: torch.Tensor | None = None) -> Accepted:
    """Walks every row's tree from node 0 to the first child whose token is the
    target's choice, until no child is or ``max_path`` (at most 64) nodes are
    walked, and moves the walked nodes' keys and values in every cache from
    places ``lengths[b] + node`` to ``lengths[b] + 0, 1, 2, ...`` (C ABI
    ``aspire_tree_accept``, one launch for up to 128 layers).

    ``tokens``, ``parents`` and ``targets`` are int32 ``[total]``, ``indptr``
    int32 ``[rows + 1]``, ``lengths`` int32 ``[rows]`` the committed tokens
    before the step.  ``caches`` are the layers' contiguous ``[pages, 2,
    page_size, heads, head_dim]`` tensors of one shape, changed in place
    through ``block_table`` int32 ``[rows, columns]``.

    ``kv_len`` int32 ``[rows]`` are the step's keys of each row, as
    :func:`aspire_b200.kv_ops.build_step_tables` gives them: a row that got no
    pages has 0 and commits nothing, its length stays, and a later step may
    serve it.  The walk then also ends before a node whose place has no page.
    Without ``kv_len`` the keys of all nodes are taken to be in the cache.

    A negative target is no token (``pick_tokens`` gives -1 where nothing is
    allowed) and no draft's: the walk ends before its node, which stays the
    row's last committed token and so the root of its next tree, and
    ``status`` gets ``ASPIRE_STATUS_NO_TOKEN``."""
    return Accepted(*_capi.ops().tree_accept(tokens, parents, targets, indptr, lengths, max_path, caches, block_table,
                                             status, kv_len))
