"""What a step with drafted trees does behind the model (speculative decoding): the walk along the sampled tokens, and the
accepted nodes' cache rows to their places.  Both run on the GPU without a look at their results, so the next step can
be prepared from them (engine/block_tables.py) before the host knows what was accepted.

One step, with `state` a DeviceBlockTables and node 0 of each tree the last token that was committed:

    t = state.step(rows, cached_lens, tree_lens, num_tokens, parents, mask_words)
    set_tree_context(t.cu_seqlens_q, t.context_lens, t.slot_mapping, t.block_tables, t.tree_masks)
    logits = model(draft_tokens, t.positions)                       # Attention.forward stores and attends
    target_tokens = sampler(logits)                                 # one sample behind every node
    a = accept_tree(draft_tokens, target_tokens, parents, t.cu_seqlens_q, cached_lens, t.context_lens, max_path)
    compact_kvcache(kv_cache, a.path, a.accepted, cached_lens, t.block_tables)
    state.release(rows, a.cached_lens)                              # blocks that only rejected nodes had
    # a.tokens[:, :accepted] are the step's tokens; the last of them is the root of the next tree
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _lib


class Accepted(NamedTuple):
    """accepted (sequences) nodes on each path, path (sequences, max_path) their indices within the tree, tokens (sequences,
    max_path; int64) what the target model sampled behind them, both -1 behind the last; cached_lens: the lengths that the
    cache holds once the rows have been moved."""
    accepted: torch.Tensor
    path: torch.Tensor
    tokens: torch.Tensor
    cached_lens: torch.Tensor


def accept_tree(draft_tokens, target_tokens, parents, cu_seqlens_q, cached_lens, context_lens, max_path: int) -> Accepted:
    """From the root on to the (first) child whose draft token is what the target model sampled behind its parent.  Details:
    b200_accept_tree in include/b200_attn.h."""
    return Accepted(*_lib.native().accept_tree(draft_tokens, target_tokens, parents, cu_seqlens_q, cached_lens, context_lens, max_path))


def compact_kvcache(kv_cache, path, accepted, start_lens, block_tables):
    """In every plane of kv_cache (..., blocks, block size, kv heads, head_dim) the row of position start_lens[i] +
    path[i, k] goes to start_lens[i] + k, k < accepted[i].  Details: b200_compact_kvcache in include/b200_attn.h."""
    _lib.native().compact_kvcache(kv_cache, path, accepted, start_lens, block_tables)
