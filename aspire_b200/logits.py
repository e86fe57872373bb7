"""Penalties for repeated tokens, biases and grammar masks on a step's logits.

For token v of a step's token t, with c occurrences of v in the row's history
behind its prompt and among the step's tokens on t's path::

    x = x / repetition  if x > 0 else  x * repetition     v in the history or on the path
    x = x - frequency * c - presence * (c > 0)
    x = x + bias[v]
    x = -inf                                              v not allowed

in fp32, each operation rounded on its own, rounded to the logits' type once
at the end (C ABI ``aspire_adjust_logits``).  The calls have no gradient.
"""

from __future__ import annotations

import torch

from . import _capi

_Bias = tuple[torch.Tensor, torch.Tensor, torch.Tensor]


def _call(logits, history, history_len, prompt_len, indptr, tokens, tree_mask, repetition, frequency, presence, bias,
          allowed, out, want_out, want_ids, status):
    at, ids, values = bias if bias is not None else (None, None, None)
    return _capi.ops().adjust_logits(logits, history, history_len, prompt_len, indptr, tokens, tree_mask, repetition,
                                     frequency, presence, at, ids, values, allowed, out, want_out, want_ids, status)


def adjust_logits(logits: torch.Tensor, *, history: torch.Tensor | None = None,
                  history_len: torch.Tensor | None = None, prompt_len: torch.Tensor | None = None,
                  indptr: torch.Tensor | None = None, tokens: torch.Tensor | None = None,
                  tree_mask: torch.Tensor | None = None, repetition: torch.Tensor | None = None,
                  frequency: torch.Tensor | None = None, presence: torch.Tensor | None = None,
                  bias: _Bias | None = None, allowed: torch.Tensor | None = None, out: torch.Tensor | None = None,
                  status: torch.Tensor | None = None) -> torch.Tensor:
    """The adjusted ``logits`` ``[tokens, vocab]`` (fp32, bf16 or fp16).

    ``indptr`` int32 ``[rows + 1]``: the rows' tokens; without it each token is
    a row of its own.  ``history`` int32 ``[rows, columns]`` holds
    ``history_len`` int32 ``[rows]`` tokens before the step's, the first
    ``prompt_len`` int32 ``[rows]`` of them the prompt, which only the
    repetition penalty counts.  ``tokens`` int32 ``[tokens]`` are the step's
    own: on a token's path lie those that its ``tree_mask`` int32 ``[tokens,
    words]`` names (as :func:`aspire_b200.kv_ops.build_step_tables` makes it)
    or, without masks, those of its row up to itself.  ``repetition``,
    ``frequency`` and ``presence`` are fp32 ``[rows]``; ``bias`` is ``(indptr
    int32 [rows + 1], ids int32, values fp32)``, of a token listed twice the
    later value; ``allowed`` int32 ``[tokens, vocab / 32 rounded up]`` has bit
    v % 32 of word v / 32 set where v may follow.  Token ids outside ``[0,
    vocab)`` are ignored.  ``out`` may be ``logits`` itself.  Tokens of no row
    keep their logits."""
    return _call(logits, history, history_len, prompt_len, indptr, tokens, tree_mask, repetition, frequency, presence,
                 bias, allowed, out, True, False, status)[0]


def pick_tokens(logits: torch.Tensor, *, history: torch.Tensor | None = None,
                history_len: torch.Tensor | None = None, prompt_len: torch.Tensor | None = None,
                indptr: torch.Tensor | None = None, tokens: torch.Tensor | None = None,
                tree_mask: torch.Tensor | None = None, repetition: torch.Tensor | None = None,
                frequency: torch.Tensor | None = None, presence: torch.Tensor | None = None,
                bias: _Bias | None = None, allowed: torch.Tensor | None = None,
                status: torch.Tensor | None = None) -> torch.Tensor:
    """The best token int32 ``[tokens]`` of the adjusted logits (arguments as
    for :func:`adjust_logits`), which are not written: the largest value before
    its rounding, the lowest id on ties.  NaN and -inf are never chosen; -1
    where nothing else is left, and for tokens of no row."""
    return _call(logits, history, history_len, prompt_len, indptr, tokens, tree_mask, repetition, frequency, presence,
                 bias, allowed, None, False, True, status)[1]
