"""Packed (varlen) batch description shared by models, engine and ops."""
from __future__ import annotations

from dataclasses import dataclass
from typing import List, Optional, Sequence

import torch


@dataclass
class SharedPrefix:
    """Groups of sequences that begin with the same cached tokens: attention reads those once per group.

    Group j holds the sequences first[j] .. first[j + 1] - 1 of the batch; their first lens[j] tokens lie in the pages block_tables[j] (0: nothing
    is shared).  The sequences' own block tables name the same pages at their front and their lengths count the shared tokens.  Sequences outside
    of first[0] .. first[-1] have no shared part.  ``max_len`` and ``max_rows`` bound lens and the query rows of a group that shares something; the
    tensors may change under them, as in a captured step."""
    block_tables: torch.Tensor  # [G, max_blocks] int32
    lens: torch.Tensor          # [G] int32
    first: torch.Tensor         # [G + 1] int32, ascending
    num_groups: int
    max_len: int
    max_rows: int

    @staticmethod
    def build(groups: Sequence[Sequence[int]], block_tables: Sequence[Sequence[int]], lens: Sequence[int], q_lens: Sequence[int],
              device) -> Optional["SharedPrefix"]:
        """``groups``: sequence numbers of each group, consecutive and ascending; ``block_tables`` / ``lens``: a group's shared pages and tokens;
        ``q_lens``: query rows of every sequence of the batch.  None where nothing is shared."""
        if not groups or max(lens) == 0:
            return None
        flat = [i for g in groups for i in g]
        if flat != list(range(flat[0], flat[0] + len(flat))) or not all(groups):
            raise ValueError(f"SharedPrefix: groups of consecutive sequences, got {list(groups)}")
        width = max(1, max(len(t) for t in block_tables))
        i32 = dict(dtype=torch.int32)
        return SharedPrefix(
            block_tables=torch.tensor([list(t) + [0] * (width - len(t)) for t in block_tables], **i32).to(device),
            lens=torch.tensor(list(lens), **i32).to(device),
            first=torch.tensor([g[0] for g in groups] + [groups[-1][-1] + 1], **i32).to(device), num_groups=len(groups), max_len=max(lens),
            max_rows=max(sum(q_lens[i] for i in g) for g in groups))


@dataclass
class DraftTree:
    """The new tokens of every sequence of a batch as a tree of guesses (``ops.step_layout`` makes the masks).

    ``parents``: a token's parent by its place among its sequence's new tokens, -1 for none, parents before children.  ``masks``: bit j of a row: it sees
    its sequence's new token j; attention goes by these alone."""
    parents: torch.Tensor       # [T] int32
    masks: torch.Tensor         # [T, words] int32


@dataclass
class BatchInput:
    tokens: torch.Tensor        # [T] int32 token ids, sequences packed back to back
    positions: torch.Tensor     # [T] int32 absolute position of each token
    slot_mapping: torch.Tensor  # [T] int32 KV-cache slot (block * block_size + offset); < 0 = do not write
    block_tables: torch.Tensor  # [B, max_blocks] int32
    seq_lens: torch.Tensor      # [B] int32 total cached length *including* this step's tokens
    cu_q: torch.Tensor          # [B + 1] int32 query row offsets
    last_idx: torch.Tensor      # [B] int64 row of the last token of each sequence
    num_seqs: int
    max_q: int
    max_kv: int
    is_decode: bool             # exactly one query token per sequence
    is_fresh_prefill: bool      # no sequence has prior context (seq_len == q_len)
    decode_splits: int = 0      # split-KV factor frozen at graph-capture time (0 = choose per call)
    state_slots: Optional[torch.Tensor] = None   # [B] int32 state slot of each sequence (recurrent models); < 0 = inert row
    prefix: Optional[SharedPrefix] = None        # cached tokens that groups of sequences share
    tree: Optional[DraftTree] = None             # new tokens are trees of guesses

    @staticmethod
    def build(token_lists: Sequence[Sequence[int]], context_lens: Sequence[int], block_tables: Sequence[Sequence[int]],
              block_size: int, device, max_blocks: Optional[int] = None, pad_to: int = 1,
              state_slots: Optional[Sequence[int]] = None, parents: Optional[Sequence[Sequence[int]]] = None) -> "BatchInput":
        """``token_lists[i]`` are the new tokens of sequence i, which already has ``context_lens[i]`` tokens in the cache blocks ``block_tables[i]``;
        ``parents[i]``: they are a tree (DraftTree).  Goes to the device as one upload, what follows from the lengths is formed there."""
        from ..ops import step_layout

        q_lens = [len(t) for t in token_lists]
        for n, ctx, bt in zip(q_lens, context_lens, block_tables):
            if ctx + n > len(bt) * block_size and n:
                raise IndexError(f"{ctx} + {n} tokens in {len(bt)} blocks of {block_size}")
        B, T, counts = len(q_lens), sum(q_lens), [len(b) for b in block_tables]
        mb = max_blocks or max(1, max(counts))
        if max(counts, default=0) > mb:
            raise ValueError(f"{max(counts)} blocks in a table of {mb}")
        # inert padding rows (token 0, slot -1, owned by no sequence) so that the packed length is a
        # multiple of `pad_to` (sequence-parallel prefill shards the rows evenly over the ranks)
        rows = T + -T % pad_to
        parts = [[x for t in token_lists for x in t] + [0] * (rows - T), list(context_lens), q_lens, counts, [b for bt in block_tables for b in bt]]
        if parents is not None:
            if [len(p) for p in parents] != q_lens:
                raise ValueError(f"trees of {[len(p) for p in parents]} parents for {q_lens} tokens")
            parts.append([x for p in parents for x in p] + [-1] * (rows - T))
        if state_slots is not None:
            parts.append(list(state_slots))
        sizes = [len(p) for p in parts]
        parts = list(torch.tensor([int(x) for p in parts for x in p], dtype=torch.int32).to(device).split(sizes))
        tokens, context, new, counts, pages = parts[:5]
        max_q = max(q_lens, default=0)
        up = parts[5] if parents is not None else None
        at = step_layout(context, new, pages, block_size, rows, max_q, page_counts=counts, max_blocks=mb, parents=up)
        return BatchInput(
            tokens=tokens, positions=at.positions, slot_mapping=at.slot_mapping, block_tables=at.block_tables, seq_lens=at.seq_lens, cu_q=at.cu_q,
            last_idx=at.last_idx, num_seqs=B, max_q=max_q, max_kv=max((c + n for c, n in zip(context_lens, q_lens)), default=0),
            is_decode=all(q == 1 for q in q_lens), is_fresh_prefill=all(c == 0 for c in context_lens),
            state_slots=None if state_slots is None else parts[-1], tree=None if up is None else DraftTree(parents=up, masks=at.masks))
