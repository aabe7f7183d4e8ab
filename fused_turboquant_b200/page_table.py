"""Pages of a batch of requests, kept on the GPU: block table, lengths and free blocks of a ``PagedKVPool``.

The reference leaves this to its engine, which keeps block tables on the host and copies them over at every
step.  Here a step's table and slot map come out of one launch from the requests' lengths, without a host
synchronisation, so that a step can be captured in a CUDA graph.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib


class Extension(NamedTuple):
    """What ``PageTable.extend`` gave: ``slots`` int64, ``granted`` int32 [R] (tokens, all of a request's or
    none: of a drafted tree the ``tree_lens`` of the calls that follow), ``starts`` int32 [R + 1] (place of a request's first token in the flat slot map)."""
    slots: torch.Tensor
    granted: torch.Tensor
    starts: torch.Tensor


class PageTable:
    """``block_table`` int32 [max_requests, max_blocks] (-1: no block), ``seq_lens`` int32 [max_requests],
    ``free_blocks`` int32 [num_blocks] of which the first ``n_free`` (int32 [1]) are free, the last of them
    taken first.  All four keep their memory: pass them to captured kernels as they are."""

    def __init__(self, num_blocks: int, max_requests: int, max_blocks: int, device="cuda"):
        if num_blocks < 0 or max_requests < 0 or max_blocks < 1:
            raise ValueError(f"bad page table: {num_blocks} blocks, {max_requests} requests of up to {max_blocks} blocks")
        if max_requests > 8192:
            raise ValueError(f"a page table has at most 8192 requests, got {max_requests}")
        if torch.device(device).type != "cuda":
            raise RuntimeError("a page table lives on a CUDA device: fused_turboquant_b200 has no CPU path")
        self.num_blocks, self.max_requests, self.max_blocks = num_blocks, max_requests, max_blocks
        opts = dict(dtype=torch.int32, device=device)
        self.block_table = torch.full((max_requests, max_blocks), -1, **opts)
        self.seq_lens = torch.zeros(max_requests, **opts)
        self.free_blocks = torch.arange(num_blocks - 1, -1, -1, **opts)
        self.n_free = torch.full((1,), num_blocks, **opts)

    def extend(self, new_lens: torch.Tensor, width: int, packed: bool = False) -> Extension:
        """Room for ``new_lens[r]`` more tokens of every request.

        A request gets all its tokens or none: none where they do not fit its row of the table or ``width``, where
        the number is negative, or where it needs blocks and the needs of the requests up to it exceed the free ones.
        ``slots`` is [R, width] (a row per request, -1 behind its tokens) or, ``packed``, [width] with the requests'
        tokens back to back: ``starts`` says where each begins.
        """
        return Extension(*_lib.native().pages_extend(self.block_table, self.seq_lens, self.free_blocks, self.n_free,
                                                     new_lens, width, packed))

    def trim(self, keep_lens: torch.Tensor) -> None:
        """Requests keep their first ``keep_lens[r]`` tokens (no more than they have; 0 ends a request); blocks
        without a token are free again."""
        _lib.native().pages_trim(self.block_table, self.seq_lens, self.free_blocks, self.n_free, keep_lens)

    def state_dict(self) -> dict:
        """The four tensors themselves, not copies."""
        return dict(block_table=self.block_table, seq_lens=self.seq_lens, free_blocks=self.free_blocks, n_free=self.n_free)

    def load_state_dict(self, state: dict) -> None:
        """Copies another table's state into this one's memory (same sizes)."""
        for name, mine in self.state_dict().items():
            if state[name].shape != mine.shape:
                raise ValueError(f"{name} is {tuple(state[name].shape)}, this table's is {tuple(mine.shape)}")
        for name, mine in self.state_dict().items():
            mine.copy_(state[name])
