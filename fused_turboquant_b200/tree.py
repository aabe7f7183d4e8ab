"""Trees of drafted tokens: ancestor masks and positions.

A tree of ``n_nodes`` tokens is given by ``parents`` [B, n_nodes]: a node's parent has a lower index; anything else
(-1) makes it a root.  Node 0 is the token that the last step ended with.  The reference verifies drafts as chains
only (vllm_plugin/v1_backend.py:1359-1384).  Attention over a tree is ``PagedKVPool.tree_attention``, what happens to
it afterwards ``PagedKVPool.tree_commit``.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

MAX_NODES = 256


class Accepted(NamedTuple):
    """What ``PagedKVPool.tree_commit`` accepted: ``path`` int32 [B, n_nodes] (nodes from the root on, then -1),
    ``n_accepted`` int32 [B], ``tokens`` int32 [B, n_nodes] (the step's new tokens, then -1), ``seq_lens`` int32 [B]
    (context + accepted)."""
    path: torch.Tensor
    n_accepted: torch.Tensor
    tokens: torch.Tensor
    seq_lens: torch.Tensor


def ancestor_masks(parents: torch.Tensor, tree_lens: torch.Tensor | None = None,
                   context_lens: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(masks int32 [B, n_nodes, ceil(n_nodes / 32)], positions int32 [B, n_nodes]).

    Bit j % 32 of word j // 32 of a node's mask: node j is the node itself or one of its ancestors.  A node's
    position is ``context_lens[b]`` (0 without it) plus its depth.  Nodes from ``tree_lens[b]`` on do not exist: their
    masks are empty.
    """
    return _lib.native().tree_masks(parents, tree_lens, context_lens)
