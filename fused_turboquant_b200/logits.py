"""Logits of a serving step: penalties for repeated tokens, biases, grammar masks, the best token.

One pass over the logits; the tokens that a request has seen are counted on the fly (no [requests, vocabulary] table
of counts exists), and with a drafted tree every node's logits are penalised for the tokens on its own path.
No counterpart in the reference, which leaves sampling to its engine.
"""
from __future__ import annotations

import torch

from . import _lib


def workspace_bytes(n_rows: int, vocab: int) -> int:
    """Bytes of scratch memory of a ``process`` call of so many rows of logits that returns the best tokens."""
    return int(_lib.load().ftq_logits_workspace_bytes(n_rows, vocab))


def process(logits: torch.Tensor, *, history: torch.Tensor | None = None, history_lens: torch.Tensor | None = None,
            prompt_lens: torch.Tensor | None = None, repetition: torch.Tensor | None = None,
            frequency: torch.Tensor | None = None, presence: torch.Tensor | None = None,
            bias_ids: torch.Tensor | None = None, bias: torch.Tensor | None = None,
            allowed: torch.Tensor | None = None, tree_tokens: torch.Tensor | None = None,
            tree_masks: torch.Tensor | None = None, out: torch.Tensor | None = None, return_logits: bool = True,
            return_best: bool = True, workspace: torch.Tensor | None = None):
    """(processed logits fp32 of the logits' shape, best token int32 per row); None for what is not returned.

    logits: [R, V] or [R, rows, V] (a row per node of a drafted tree), fp32 / fp16 / bf16.
    history [R, H], history_lens [R]: a request's tokens so far, the first ``prompt_lens[r]`` of them its prompt and the
    others its answer.  tree_tokens [R, rows], tree_masks [R, rows, ceil(rows / 32)]: the tokens of the nodes in a
    row's mask count as answer too (so the history ends before the tree's root).
    In this order, each rounded once in fp32:
      repetition [R]: x / p where x > 0, else x * p, for tokens of the prompt or the answer;
      frequency [R]: minus p * (times in the answer);  presence [R]: minus p for tokens of the answer;
      bias [R, K] added at bias_ids [R, K] (negative: unused; of equal ids the last);
      allowed [R, rows, ceil(V / 32)] int32 words: -inf where the token's bit (v % 32 of word v // 32) is clear.
    The best token is the lowest index of the largest value (NaN above all); it takes scratch memory (``workspace_bytes``), which
    calls on the same stream share unless it is passed in: a captured graph that runs beside others needs its own.  ``out`` may be
    ``logits`` itself where that is dense fp32.
    """
    if out is None and not return_logits and not return_best:
        raise ValueError("nothing to return")
    return _lib.native().logits_process(logits, history, history_lens, prompt_lens, repetition, frequency, presence,
                                        bias_ids, bias, allowed, tree_tokens, tree_masks, out, return_logits, return_best, workspace)
