"""Steps that check drafted tokens: what ``ops.step_layout`` and ``ops.accept_drafts`` return, and what they ask of their arguments.

A tree of drafts: a sequence's new tokens are its last sampled one (token 0, whose place in the cache is still empty) and guesses for what follows it, each
behind its parent.  All of them go through the model in one step, each seeing the cached tokens, its ancestors and itself; a sample drawn at every
one of them says which path is right.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

MAX_TREE = 1024            # tokens of a tree: 32 words of mask


class StepLayout(NamedTuple):
    positions: torch.Tensor               # [rows] int32
    slot_mapping: torch.Tensor            # [rows] int32
    seq_lens: torch.Tensor                # [B] int32
    cu_q: torch.Tensor                    # [B + 1] int32
    last_idx: torch.Tensor                # [B] int64
    block_tables: torch.Tensor            # [B, max_blocks] int32
    masks: Optional[torch.Tensor]         # [rows, words] int32, of trees


class Accepted(NamedTuple):
    tokens: torch.Tensor                  # [B, max_q] int32: what was sampled along the path, -1 behind it
    counts: torch.Tensor                  # [B] int32: how many
    path: torch.Tensor                    # [B, max_q] int32: the path's places among a sequence's new tokens, -1 behind it
    context_lens: torch.Tensor            # [B] int32: cached tokens, the path's included


def wrong_ints(dev: int, *tensors) -> bool:
    """Whether one of the tensors is not contiguous int32 on device ``dev``."""
    for t in tensors:
        if t.dtype is not torch.int32 or not t.is_contiguous() or t.get_device() != dev:
            return True
    return False


def check_layout(context_lens, new_lens, pages, page_size, rows, max_new, page_counts, max_blocks, parents):
    """(sequences, columns of the block tables, words of a mask)"""
    dev, B = context_lens.get_device(), context_lens.numel()
    if wrong_ints(dev, context_lens, new_lens, pages) or new_lens.numel() != B:
        raise ValueError(f"step_layout: context_lens, new_lens and pages are contiguous int32 on one device, lengths of the same {B} sequences")
    if page_size <= 0 or rows < 0 or max_new < 0:
        raise ValueError(f"step_layout: pages of {page_size} tokens, {rows} rows, up to {max_new} new tokens")
    if page_counts is not None:
        if wrong_ints(dev, page_counts) or page_counts.numel() != B or pages.dim() != 1 or max_blocks is None or max_blocks < 0:
            raise ValueError(f"step_layout: lists of pages are one list back to back, with int32 page_counts of {B} sequences and max_blocks")
    else:
        if pages.dim() != 2 or pages.shape[0] < B or max_blocks not in (None, pages.shape[1]):
            raise ValueError(f"step_layout: without page_counts, pages are block tables of {B} sequences or more, got {tuple(pages.shape)}")
        max_blocks = pages.shape[1]
    words = 0
    if parents is not None:
        if wrong_ints(dev, parents) or parents.numel() < rows:
            raise ValueError(f"step_layout: parents are contiguous int32 on the lengths' device, {rows} or more")
        if max_new > MAX_TREE:
            raise ValueError(f"step_layout: trees of up to {MAX_TREE} tokens, got {max_new}")
        words = -(-max_new // 32)
    return B, max_blocks, words


def check_accept(sampled, batch, pages):
    """(planes, blocks, heads, page size) of the cache tensors, (0, 0, 1, 1) without one"""
    if batch.tree is None:
        raise ValueError("accept_drafts: the batch has no tree")
    dev, parents, B = sampled.get_device(), batch.tree.parents, batch.num_seqs
    T = parents.numel()
    if wrong_ints(dev, sampled, batch.tokens, parents, batch.cu_q, batch.seq_lens, batch.block_tables) or sampled.numel() < T or batch.tokens.numel() < T:
        raise ValueError(f"accept_drafts: sampled, tokens, parents, cu_q, seq_lens and block_tables are contiguous int32 on one device, {T} rows or more")
    if batch.cu_q.numel() < B + 1 or batch.seq_lens.numel() < B or batch.block_tables.dim() != 2 or batch.block_tables.shape[0] < B:
        raise ValueError(f"accept_drafts: cu_q, seq_lens and block_tables of {B} sequences or more")
    if batch.max_q > MAX_TREE:
        raise ValueError(f"accept_drafts: trees of up to {MAX_TREE} tokens, got {batch.max_q}")
    if not pages:
        return 0, 0, 1, 1
    lead = pages[0].shape[:-1]
    n = len(lead)
    if n < 3:
        raise ValueError(f"accept_drafts: cache tensors are [.., blocks, heads, block_size, d], got {tuple(pages[0].shape)}")
    for x in pages:
        if x.shape[:n] != lead or not x.is_contiguous() or x.get_device() != dev or (x.numel() == 0 and lead.numel() > 0):
            raise ValueError(f"accept_drafts: cache tensors are contiguous, on {sampled.device}, and alike up to a row ({tuple(lead)}), got {tuple(x.shape)} "
                             f"on {x.device}")
    return lead[:-3].numel(), lead[-3], lead[-2], lead[-1]
