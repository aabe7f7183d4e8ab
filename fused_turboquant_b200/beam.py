"""Beam search: the best continuations over beams and vocabulary.

A step of a request with K beams: ``logits.process`` for penalties and masks where they are wanted, ``select`` for the
continuations, ``PageTable.fork`` for the beams' rows of the block table (``PagedKVPool.copy_pages`` for their caches),
``PageTable.extend`` and ``PagedKVPool.store`` for the next token, ``PagedKVPool.shared_attention`` for its attention.
No counterpart in the reference, which leaves decoding to its engine.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .kernels import _DT

MAX_BEAMS = 64          # and continuations selected for a request
MAX_END_TOKENS = 16


class Selection(NamedTuple):
    """What ``select`` chose: ``scores`` fp32, ``parents`` and ``tokens`` int32, [R, n_best] each, the best first (where there are
    fewer: -inf, -1, -1), and ``end_scores`` fp32 [R, K, n] (None without end tokens)."""
    scores: torch.Tensor
    parents: torch.Tensor
    tokens: torch.Tensor
    end_scores: torch.Tensor | None


def workspace_bytes(dtype: torch.dtype, requests: int, beams: int, vocab: int, n_best: int, n_end_tokens: int = 0) -> int:
    """Bytes of scratch memory of a ``select`` call (0: no such call)."""
    return int(_lib.load().ftq_beam_workspace_bytes(_DT.get(dtype, -1), requests, beams, vocab, n_best, n_end_tokens))


def select(logits: torch.Tensor, scores: torch.Tensor, n_best: int, *, end_tokens: torch.Tensor | None = None,
           workspace: torch.Tensor | None = None) -> Selection:
    """The ``n_best`` best continuations of every request.

    logits: [R, K, V], fp32 / fp16 / bf16, up to 65535 requests; scores: [R, K], the beams' log-probabilities so far, -inf for a
    beam that is not alive (of which at the first step of a request all but one are: they would all say the same).  Token v after beam b scores
    ``scores[b] + log_softmax(logits[b])[v]``; of equal ones the lowest beam's lowest token comes first.  Totals are compared in 64
    bits, but the sums of exponentials in them are fp32's: totals of different beams that lie within some 1e-7 may come in either
    order, those of beams with the same logits and scores are equal.
    ``end_tokens`` [n] end an answer: they are not selected, and ``end_scores`` says what each beam would score with each of them.
    A beam whose logits hold a NaN or +inf, or nothing but -inf, has no continuation.

    ``parents`` [R, K] of ``n_best`` = K beams go to ``PageTable.fork``.  No host synchronisation; graph-capturable.  Scratch
    memory (``workspace_bytes``) is shared by the calls on the same stream unless it is passed in: a captured graph that runs
    beside others needs its own.
    """
    return Selection(*_lib.native().beam_select(logits, scores, n_best, end_tokens, workspace))
