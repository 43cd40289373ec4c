"""The structure of a flat batch - offsets, positions, block table, slot map - from request lengths (csrc/batch_plan.cu)."""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _lib
from .core import _launch

P, I, L = C.c_void_p, C.c_int, C.c_longlong
_SIGS = {
    "sllm_batch_plan": (I, [P, P, P, L, I, I, I, L, I, P, P, P, P, P, P, P, P]),
}


_lib.EXTRA_KERNEL_SIGNATURES.update(_SIGS)
_k = _lib.kernels
MAX_REQUESTS = 16384           # whose running sums fit in shared memory
MAX_COUNT = 2 ** 31 - 4096


class BatchPlan(NamedTuple):
    """What a `ForwardBatch` consists of beside its tokens, for S requests in T rows."""
    row_off: torch.Tensor          # int32 [S + 1]: rows of request s are row_off[s] .. row_off[s + 1]
    positions: torch.Tensor        # int32 [T], -1 behind the last request
    seq_index: torch.Tensor        # int32 [T], -1 behind the last request
    kv_lens: torch.Tensor          # int32 [T]: position + 1, 0 behind the last request
    slots: torch.Tensor            # int64 [T]: page * page_size + place of the row's key and value, -1 behind the last request
    last_rows: torch.Tensor        # int64 [S], -1 of a request without new tokens
    block_table: torch.Tensor      # int32 [S, max_blocks]: a request's pages, then zeros


def _cpu(new, starts, pages, rows, max_blocks, page, table):
    new, starts = new.long().clamp(min=0), starts.long().clamp(min=0)
    s = new.numel()
    count = (starts + new + page - 1) // page
    row_off = torch.cat([new.new_zeros(1), torch.cumsum(new, 0)])
    first = torch.cumsum(count, 0) - count
    listed = torch.cat([pages.long(), pages.new_zeros(1, dtype=torch.int64)])
    page_at = lambda i: listed[i.clamp(max=pages.numel())]
    seq = torch.repeat_interleave(torch.arange(s), new)[:rows]
    pos = starts[seq] + torch.arange(seq.numel()) - row_off[seq]
    fill = lambda v, n: torch.cat([v, torch.full((rows - v.numel(),), n, dtype=torch.int64)])
    slots = page_at(first[seq] + pos // page) * page + pos % page
    col = torch.arange(max_blocks)
    table.copy_(torch.where(col < count[:, None], page_at(first[:, None] + col), 0))
    i32 = lambda t: t.to(torch.int32)
    return BatchPlan(i32(row_off), i32(fill(pos, -1)), i32(fill(seq, -1)), i32(fill(pos + 1, 0)), fill(slots, -1),
                     torch.where(new > 0, row_off[1:] - 1, -1), table)


def batch_plan(new_lens: torch.Tensor, starts: torch.Tensor, pages: torch.Tensor, rows: int, max_blocks: int, page_size: int = 16,
               table: Optional[torch.Tensor] = None) -> BatchPlan:
    """The plan of requests with ``new_lens`` [S] tokens each behind ``starts`` [S] tokens that their pages hold already (int32).
    ``pages`` (int32): the requests' pages one after another, ceil((starts + new_lens) / page_size) of each.  ``rows``: rows of the
    batch, the sum of new_lens or more (a captured step's padding).  ``table`` (int32 [S, max_blocks], any row stride) receives
    the block table in place of a new tensor.  A length below 0 counts as 0; entries whose page lies beyond the list read page 0, and
    a table narrower than a request holds its first pages.  Positions stay below 2^31, requests at 16384 or less."""
    s, dev = new_lens.numel(), new_lens.device
    for t in (new_lens, starts, pages):
        if t.dtype is not torch.int32 or t.dim() != 1 or t.device != dev or not t.is_contiguous():
            raise ValueError("lengths, starts and pages are contiguous int32 vectors on one device")
    if starts.numel() != s:
        raise ValueError("one start per length")
    if s > MAX_REQUESTS:
        raise ValueError(f"at most {MAX_REQUESTS} requests")
    if not 0 <= rows <= MAX_COUNT or not 0 <= max_blocks <= MAX_COUNT or not 1 <= page_size < 2 ** 31 or pages.numel() >= 2 ** 31:
        raise ValueError("rows, max_blocks, page_size and pages are counts below 2^31")
    if table is not None and (table.dtype != torch.int32 or table.shape != (s, max_blocks) or table.device != dev
                              or (max_blocks > 1 and table.stride(1) != 1) or (s > 1 and table.stride(0) < max_blocks)):
        raise ValueError("the table is int32 [requests, max_blocks] with contiguous rows that do not overlap")
    if _lib.on_cpu(new_lens):
        return _cpu(new_lens, starts, pages, rows, max_blocks, page_size,
                    torch.empty((s, max_blocks), dtype=torch.int32) if table is None else table)
    # (one allocation, every part of it at a multiple of 16 bytes: a tensor of its own for each costs more than the kernel)
    row4 = (rows + 3) & -4
    off_at = 0 if table is not None else (s * max_blocks + 3) & -4
    pos_at = off_at + ((s + 4) & -4)
    slot_at = (pos_at + 3 * row4) // 2
    last_at = slot_at + ((rows + 1) & -2)
    out64 = torch.empty(last_at + s, dtype=torch.int64, device=dev)
    out = out64.view(torch.int32)
    if table is None:
        table = out.as_strided((s, max_blocks), (max_blocks, 1), 0)
    row_off = out.as_strided((s + 1,), (1,), off_at)
    positions = out.as_strided((rows,), (1,), pos_at)
    seq_index = out.as_strided((rows,), (1,), pos_at + row4)
    kv_lens = out.as_strided((rows,), (1,), pos_at + 2 * row4)
    slots = out64.as_strided((rows,), (1,), slot_at)
    last_rows = out64.as_strided((s,), (1,), last_at)
    rc = _launch(dev, _k().sllm_batch_plan, new_lens.data_ptr(), starts.data_ptr(), pages.data_ptr(), pages.numel(), s, rows, max_blocks,
                 table.stride(0) if s > 1 else max_blocks, page_size, row_off.data_ptr(), positions.data_ptr(), seq_index.data_ptr(),
                 kv_lens.data_ptr(), slots.data_ptr(), last_rows.data_ptr(), table.data_ptr())
    _lib.check(rc, "batch_plan")
    return BatchPlan(row_off, positions, seq_index, kv_lens, slots, last_rows, table)
