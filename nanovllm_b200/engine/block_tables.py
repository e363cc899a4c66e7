"""Block tables, slots and positions of a step built on the GPU from request lengths.

nano-vllm's BlockManager hands out blocks in Python (nanovllm/engine/block_manager.py:26-112) and its model runner
prepares a step on the host (nanovllm/engine/model_runner.py:119-179).  That needs the lengths on the host; with drafted
trees they come out of a walk on the GPU (engine/tree_decode.py).  `DeviceBlockTables` keeps the free list and every
request's block table on the GPU: `step()` is one launch from lengths to all that a step's kernels read, `release()`
gives blocks back.  Neither synchronises, and both can be captured into a CUDA graph.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _lib


class StepTables(NamedTuple):
    """What a step's kernels read.  cu_seqlens_q, cu_seqlens_k (sequences + 1), context_lens (sequences), slot_mapping and
    positions (tokens; int32 and int64), block_tables (sequences, columns; -1 behind the last block), tree_masks (tokens,
    words; int64; None without trees)."""
    cu_seqlens_q: torch.Tensor
    cu_seqlens_k: torch.Tensor
    context_lens: torch.Tensor
    slot_mapping: torch.Tensor
    positions: torch.Tensor
    block_tables: torch.Tensor
    tree_masks: torch.Tensor | None


class DeviceBlockTables:
    """State, all int32 on one GPU and free for the caller to read or set between steps: `tables` (requests, columns) block
    ids of each request, `owned` (requests) how many of them are its own, `free_blocks` (blocks of the cache) a stack of
    free ids of which the first pool[0] count, `pool` (2): that number, and how many sequences the last step left out."""

    def __init__(self, tables: torch.Tensor, owned: torch.Tensor, free_blocks: torch.Tensor, pool: torch.Tensor, block_size: int):
        self.tables, self.owned, self.free_blocks, self.pool, self.block_size = tables, owned, free_blocks, pool, block_size

    @classmethod
    def create(cls, max_requests: int, max_blocks: int, num_blocks: int, block_size: int, device="cuda"):
        """All blocks of a cache of `num_blocks` free (the lowest id is taken first), no request has any."""
        tables = torch.full((max_requests, max_blocks), -1, dtype=torch.int32, device=device)
        free = torch.arange(num_blocks - 1, -1, -1, dtype=torch.int32, device=device)
        return cls(tables, torch.zeros(max_requests, dtype=torch.int32, device=device), free,
                   torch.tensor([num_blocks, 0], dtype=torch.int32, device=device), block_size)

    def step(self, rows, cached_lens, new_lens, num_tokens: int, parents=None, mask_words: int = 0, out: StepTables | None = None) -> StepTables:
        """Sequence i is request rows[i] (None: i), with cached_lens[i] tokens in the cache and new_lens[i] in this step
        (num_tokens in all, one sequence behind the other); it takes what blocks it lacks.  parents (tokens) and mask_words
        make it a step of drafted trees: parents[t] is the index of the token's parent within its tree, and the masks say
        whom each node sees.  A sequence that cannot be served is left out: context length 0, slots -1, no blocks taken.
        `out`: write into these (graph buffers; context_lens may have more rows than there are sequences).  Details:
        b200_step_tables in include/b200_attn.h."""
        return StepTables(*_lib.native().step_tables(self.tables, self.owned, self.free_blocks, self.pool, self.block_size, rows, cached_lens,
                                                     new_lens, num_tokens, parents, mask_words, out))

    def release(self, rows, keep_lens):
        """Request rows[i] (None: i) keeps the blocks of its first keep_lens[i] tokens and gives the others back (0: all)."""
        _lib.native().release_blocks(self.tables, self.owned, self.free_blocks, self.pool, self.block_size, rows, keep_lens)
