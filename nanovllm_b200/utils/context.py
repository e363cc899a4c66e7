"""Per-step attention metadata record, field for field the reference's
nanovllm/utils/context.py:5-27 (a module-global replaced wholesale every step).

When this package is installed into a running nano-vllm (nanovllm_b200.integration), the
attention layer reads the reference's own record instead, so the engine's set_context() calls
reach it unchanged.  Standalone users (tests, benchmarks) use this copy.
"""
from dataclasses import dataclass

import torch


@dataclass
class Context:
    is_prefill: bool = False
    cu_seqlens_q: torch.Tensor | None = None
    cu_seqlens_k: torch.Tensor | None = None
    max_seqlen_q: int = 0
    max_seqlen_k: int = 0
    slot_mapping: torch.Tensor | None = None
    context_lens: torch.Tensor | None = None
    block_tables: torch.Tensor | None = None


@dataclass
class TreeContext(Context):
    """A step in which every sequence brings drafted tokens (not in the reference): sequence i's are rows cu_seqlens_q[i] ..
    cu_seqlens_q[i+1], the last of its context_lens[i] tokens; tree_masks says which of them each sees (None: a chain).
    Inside nano-vllm, put such a record where its get_context() looks (nanovllm.utils.context._CONTEXT)."""
    tree_masks: torch.Tensor | None = None


_CONTEXT = Context()


def get_context():
    return _CONTEXT


def set_context(is_prefill, cu_seqlens_q=None, cu_seqlens_k=None, max_seqlen_q=0, max_seqlen_k=0,
                slot_mapping=None, context_lens=None, block_tables=None):
    global _CONTEXT
    _CONTEXT = Context(is_prefill, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k,
                       slot_mapping, context_lens, block_tables)


def set_tree_context(cu_seqlens_q, context_lens, slot_mapping, block_tables, tree_masks=None):
    global _CONTEXT
    _CONTEXT = TreeContext(False, cu_seqlens_q=cu_seqlens_q, slot_mapping=slot_mapping, context_lens=context_lens,
                           block_tables=block_tables, tree_masks=tree_masks)


def reset_context():
    global _CONTEXT
    _CONTEXT = Context()
