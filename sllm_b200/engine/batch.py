"""The flat token batch every model forward consumes.

Per-row positions, sequence indices and key counts are part of the kernel ABI from the start, so
that requests at different positions share one launch (continuous batching) and a speculative
block is just several rows of one sequence.  The reference keeps these as per-request scalars,
which is why its batch planner was never connected (docs/plans/main-plan.md:894-904).
"""
from __future__ import annotations

from dataclasses import dataclass, field
from itertools import chain
from typing import Optional, Union

import numpy as np
import torch


@dataclass
class ForwardBatch:
    tokens: torch.Tensor        # int32 [T]
    positions: torch.Tensor     # int32 [T] absolute position of each token
    seq_index: torch.Tensor     # int32 [T] row of block_table that owns the token
    kv_lens: torch.Tensor       # int32 [T] keys visible to the token (position + 1)
    block_table: torch.Tensor   # int32 [S, max_blocks]
    logit_rows: Optional[torch.Tensor] = None  # int64 rows that need logits (None = all rows)
    max_kv: int = 0             # host-side upper bound on kv_lens, for split heuristics
    # Fresh-prompt prefill metadata (tokens of each sequence contiguous, starting at position 0):
    cu_seqlens: Optional[torch.Tensor] = None  # int32 [S + 1]
    max_seqlen: int = 0
    embeds: Optional[torch.Tensor] = None      # optional [T, d] input embeddings replacing the gather
    rope_pos3: Optional[torch.Tensor] = None   # optional int32 [3, T] temporal / height / width rotary positions
    cu_seqlens_host: Optional[list] = None     # the same offsets as a Python list (tile scheduling)
    # Recurrent-state (gated delta net) layers: rows of sequence s are row_off[s] .. row_off[s + 1], its state lives in
    # slot slots[s] of the state cache.
    row_off: Optional[torch.Tensor] = None     # int32 [S + 1]
    slots: Optional[torch.Tensor] = None       # int32 [S]
    # Host copies of the same structure, set by eager batches only (a captured decode step has one row per sequence):
    # row offsets, and the position of every sequence's first row.
    row_off_host: Optional[list] = None
    starts_host: Optional[list] = None
    plans: dict = field(default_factory=dict)  # device tables that ops derive from the structure, shared by the layers
    staged_bytes: int = 0                      # copied to the device for this batch (eager batches)

    @property
    def num_tokens(self) -> int:
        return self.tokens.numel()


@dataclass
class PageLists:
    """Pages of a batch's sequences up to their new lengths, one sequence after another (int32 CPU tensor): what the GPU makes a
    block table of ``max_blocks`` columns from."""
    pages: torch.Tensor
    max_blocks: int
    page_size: int

    def table(self, lengths: list) -> torch.Tensor:
        """The block table on the host, for sequences of these lengths."""
        out, at = torch.zeros((len(lengths), self.max_blocks), dtype=torch.int32), 0
        for row, n in zip(out, lengths):
            used = (n + self.page_size - 1) // self.page_size
            row[:used] = self.pages[at:at + used]
            at += used
        return out


def _planned_batch(prompts: list, table: Union[torch.Tensor, PageLists, None], device, starts: list, last_only: bool) -> ForwardBatch:
    """`make_prefill_batch` on a GPU: one copy of tokens, lengths and pages, and one launch for everything that follows from them
    (a prompt of 8192 tokens: positions and indexes as Python lists took several times its token list)."""
    from .. import ops
    lens = [len(p) for p in prompts]
    t, s = sum(lens), len(lens)
    paged = isinstance(table, PageLists)
    pages = table.pages.numpy() if paged else np.empty(0, np.int32)
    host = np.empty(t + 2 * s + pages.size, dtype=np.int32)
    host[:t] = np.fromiter(chain.from_iterable(prompts), dtype=np.int32, count=t)
    host[t:t + s], host[t + s:t + 2 * s], host[t + 2 * s:] = lens, starts, pages
    tokens, new, begun, listed = torch.from_numpy(host).to(device).split_with_sizes((t, s, s, pages.size))
    plan = ops.batch_plan(new, begun, listed, t, table.max_blocks if paged else 0, table.page_size if paged else 16)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    rows = None
    if last_only:       # (an empty prompt's place is the row ahead of it)
        rows = plan.last_rows if all(lens) else torch.tensor([c - 1 for c in cu[1:]], dtype=torch.int64, device=device)
    fresh = not any(starts)
    return ForwardBatch(tokens=tokens, positions=plan.positions, seq_index=plan.seq_index, kv_lens=plan.kv_lens,
                        block_table=plan.block_table if paged else table, logit_rows=rows,
                        max_kv=max((a + n for a, n in zip(starts, lens) if n), default=0), cu_seqlens=plan.row_off if fresh else None,
                        max_seqlen=max(lens, default=0), cu_seqlens_host=cu if fresh else None, row_off=plan.row_off, row_off_host=cu,
                        starts_host=list(starts), staged_bytes=host.nbytes)


def make_prefill_batch(prompts: list, block_table: Union[torch.Tensor, PageLists, None], device, start_positions: Optional[list] = None,
                       last_only: bool = True) -> ForwardBatch:
    """prompts: list of token-id lists, one per row of block_table (or `PageLists` in its place)."""
    from ..ops.plan import MAX_REQUESTS
    if torch.device(device).type == "cuda" and len(prompts) <= MAX_REQUESTS:
        return _planned_batch(prompts, block_table, device, list(start_positions) if start_positions is not None else [0] * len(prompts), last_only)
    if isinstance(block_table, PageLists):
        begun = start_positions or [0] * len(prompts)
        block_table = block_table.table([a + len(p) for a, p in zip(begun, prompts)]).to(device)
    toks, pos, sidx = [], [], []
    cu = [0]
    rows = []
    fresh = True
    for i, p in enumerate(prompts):
        s0 = 0 if start_positions is None else start_positions[i]
        fresh = fresh and s0 == 0
        toks.extend(p)
        pos.extend(range(s0, s0 + len(p)))
        sidx.extend([i] * len(p))
        cu.append(cu[-1] + len(p))
        rows.append(cu[-1] - 1)
    t = lambda x, dt=torch.int32: torch.tensor(x, dtype=dt, device=device)
    positions = t(pos)
    return ForwardBatch(
        tokens=t(toks), positions=positions, seq_index=t(sidx), kv_lens=positions + 1,
        block_table=block_table, logit_rows=t(rows, torch.int64) if last_only else None,
        max_kv=max(pos) + 1 if pos else 0, cu_seqlens=t(cu) if fresh else None,
        max_seqlen=max(len(p) for p in prompts) if prompts else 0, cu_seqlens_host=cu if fresh else None,
        row_off=t(cu), row_off_host=cu, starts_host=list(start_positions) if start_positions is not None else [0] * len(prompts))
