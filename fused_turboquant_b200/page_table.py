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


class Fork(NamedTuple):
    """What ``PageTable.fork`` did: ``copies`` int32 [R, 2], the blocks (from, to) that ``PagedKVPool.copy_pages`` copies, then
    -1; ``done`` int32 [1], 0 where there were too few free blocks and nothing has changed."""
    copies: torch.Tensor
    done: torch.Tensor


class PageTable:
    """``block_table`` int32 [max_requests, max_blocks] (-1: no block), ``seq_lens`` int32 [max_requests],
    ``free_blocks`` int32 [num_blocks] of which the first ``n_free`` (int32 [1]) are free, the last of them
    taken first.  All four keep their memory: pass them to captured kernels as they are.

    With ``sharing`` several rows may hold a block (``fork``): ``shares`` int32 [num_blocks] counts those besides the first."""

    def __init__(self, num_blocks: int, max_requests: int, max_blocks: int, device="cuda", sharing: bool = False):
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
        self.shares = torch.zeros(num_blocks, **opts) if sharing else None

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
        without a token are free again.  (Rows that may share blocks are cut by ``fork``.)"""
        if self.shares is not None:
            raise RuntimeError("rows of this table may share blocks: cut them with fork(parents, keep_lens)")
        _lib.native().pages_trim(self.block_table, self.seq_lens, self.free_blocks, self.n_free, keep_lens)

    def fork_workspace_bytes(self) -> int:
        """Bytes of scratch memory of a ``fork``; a ``compact`` takes less."""
        return int(_lib.load().ftq_pages_fork_workspace_bytes(self.max_requests, self.max_blocks, self.num_blocks))

    def fork(self, parents: torch.Tensor, keep_lens: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> Fork:
        """All rows at once become copies of others: row r the first ``keep_lens[r]`` tokens (without it all) of what row
        ``parents[r]`` was.

        parents: [max_requests] rows of the table, or [groups, rows of a group], each of its own group (``beam.select``'s
        parents); any other number ends the row.  Whole blocks are shared; of the rows that would have the same partly
        filled last block the first keeps it, and the others get blocks of their own, whose contents ``copies`` lists
        (``PagedKVPool.copy_pages``).  Blocks that no row holds any more are free again.  Where there are too few free ones nothing
        changes and ``done`` is 0; a free block for every row is always enough.  Scratch memory (``fork_workspace_bytes``)
        is shared by the calls on the same stream unless it is passed in.
        """
        if self.shares is None:
            raise RuntimeError("rows of this table share no blocks: make it with sharing=True")
        return Fork(*_lib.native().pages_fork(self.block_table, self.seq_lens, self.free_blocks, self.n_free, self.shares, parents,
                                              keep_lens, workspace))

    def compact(self, workspace: torch.Tensor | None = None) -> torch.Tensor:
        """Moves the blocks in use together: those beyond the first ``num_blocks - n_free`` go into the holes before.

        Returns ``copies`` int32 [num_blocks // 2, 2] for ``PagedKVPool.copy_pages``, (from, to) and then -1: no more than has to
        move, and no block that is written is read.  The free blocks are the last ones then, the lowest taken first.
        Scratch memory as in ``fork``.
        """
        return _lib.native().pages_compact(self.block_table, self.seq_lens, self.free_blocks, self.n_free, self.shares, workspace)

    def shared_lens(self, group: int) -> torch.Tensor:
        """int32 [max_requests // group]: of every ``group`` successive rows, the tokens in leading blocks that are whole and the
        same in all of them that have tokens (``PagedKVPool.shared_attention``)."""
        return _lib.native().pages_shared_lens(self.block_table, self.seq_lens, group)

    def state_dict(self) -> dict:
        """The four tensors themselves (``shares`` too, if it has them), not copies."""
        state = dict(block_table=self.block_table, seq_lens=self.seq_lens, free_blocks=self.free_blocks, n_free=self.n_free)
        return state if self.shares is None else dict(state, shares=self.shares)

    def load_state_dict(self, state: dict) -> None:
        """Copies another table's state into this one's memory (same sizes; a state without ``shares`` has no common blocks)."""
        if self.shares is None and "shares" in state:
            raise ValueError("rows of that table may share blocks, this one's may not")
        for name, mine in self.state_dict().items():
            if name != "shares" or name in state:
                if state[name].shape != mine.shape:
                    raise ValueError(f"{name} is {tuple(state[name].shape)}, this table's is {tuple(mine.shape)}")
        for name, mine in self.state_dict().items():
            if name in state:
                mine.copy_(state[name])
            else:
                mine.zero_()
