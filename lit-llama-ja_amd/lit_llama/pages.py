"""Block tables and slot maps of paged caches, made on the GPU from the requests' lengths (csrc/pages.hip).

A page holds PAGE_SIZES tokens of one sequence. A sequence has a slot: `table[slot]` its pages in order, `seen[slot]` its tokens.
`extend` gives the sequences of a call their new tokens: pages off the stack of free ones, and for every row of the call its
sequence, position and place in the cache (page number * page + token in the page); nothing of it comes back to the host, so a captured
step extends its sequences itself. `release` puts the pages of ended sequences back. A call that cannot be served (too few
free pages, a slot twice, ...) has no rows -- all -1, which the cache's kernels leave out -- and changes no table: `PageRows.status`.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import _hip

PAGE_SIZES = (16, 32, 64, 128, 256)
MAX_SEQUENCES = 4096  # of one call
MAX_SLOTS = 65536
NO_PAGES, BAD_CALL = 1, 2  # status bits


@dataclass
class PageRows:
    """The rows of a call (int32, on the device). M may be more than the sequences' tokens: the rest are -1. `work`: items (first row, rows,
    sequence) of at most `chunk` rows, those behind the last zero."""

    row0: torch.Tensor  # (B + 1) first row of each sequence
    item0: torch.Tensor  # (B + 1) first work item of each
    row_seq: torch.Tensor  # (M)
    pos: torch.Tensor  # (M)
    place: torch.Tensor  # (M)
    work: Optional[torch.Tensor]  # (M // chunk + B, 3)
    seen: torch.Tensor  # (B) the sequences' tokens with those of this call
    left: torch.Tensor  # (1) free pages behind it
    status: torch.Tensor  # (1) 0, or NO_PAGES / BAD_CALL: the call was left undone


def on_device(t: torch.Tensor, what: str) -> int:
    """The index of t's GPU."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{what} is no tensor")
    index = t.get_device()
    if index < 0:
        _hip.require_device(t, what)
    return index


def ints(t: torch.Tensor, what: str, dims: int, index: int) -> int:
    """Checks a contiguous int32 tensor with elements on device `index`; how many it has. (Few calls into torch: a decode step's
    wrappers take as long as its small kernels.)"""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.dim() != dims or not t.is_contiguous() or not (n := t.numel()):
        raise ValueError(f"{what} must be a contiguous int32 tensor of {dims} dimension(s) with elements")
    if t.get_device() != index:
        raise ValueError(f"{what} is on {t.device}, other operands on cuda:{index}")
    return n


def _tables(table, seen, free, nfree, slot, page) -> tuple:
    """(device, slots, pages a slot, sequences, pages)"""
    index = table.get_device() if isinstance(table, torch.Tensor) else -1
    ints(table, "table", 2, index)
    on_device(table, "table")
    slots, width = table.shape
    B, cap = ints(slot, "slot", 1, index), ints(free, "free", 1, index)
    if page not in PAGE_SIZES:
        raise ValueError(f"pages of {page} tokens: {PAGE_SIZES} are taken")
    if ints(seen, "seen", 1, index) != slots or ints(nfree, "nfree", 1, index) != 1:
        raise ValueError(f"{seen.numel()} lengths and {nfree.numel()} counts for a table of {slots} slots")
    if slots > MAX_SLOTS or B > MAX_SEQUENCES or max(width, cap) * page > 1 << 30:
        raise ValueError(f"up to {MAX_SLOTS} slots, {MAX_SEQUENCES} sequences a call and 2^30 tokens are taken, not {slots}, {B} and "
                         f"{max(width, cap) * page}")
    return index, slots, width, B, cap


def extend(table: torch.Tensor, seen: torch.Tensor, free: torch.Tensor, nfree: torch.Tensor, slot: torch.Tensor, add: Optional[torch.Tensor],
           M: int, page: int, chunk: int = 0, commit: bool = True, fault: Optional[torch.Tensor] = None) -> PageRows:
    """add[b] more tokens (None: one) for the sequence in slot[b]. M: rows there is room for. commit False: lengths and stack stay as
    they are (PageRows.seen and .left hold the new ones; the new pages stand in the table already), and a later call makes the same rows
    again. Calls on one set of tables follow one another on one stream."""
    index, slots, width, B, cap = _tables(table, seen, free, nfree, slot, page)
    if add is not None and ints(add, "add", 1, index) != B:
        raise ValueError(f"{add.numel()} counts for {B} sequences")
    if fault is not None and ints(fault, "fault", 1, index) != 1:
        raise ValueError("fault is one int32")
    if not 0 <= M <= 1 << 28 or chunk < 0:
        raise ValueError(f"{M} rows in items of {chunk}")
    n = M // chunk + B if chunk else 0
    if n > 1 << 28:
        raise ValueError(f"{n} work items")
    o = table.new_empty(3 * M + 3 * n + 3 * B + 4)
    row_seq, pos, place, work, row0, item0, after, left, status = o.split_with_sizes([M, M, M, 3 * n, B + 1, B + 1, B, 1, 1])
    rows = o.data_ptr()
    items = rows + 12 * M
    tail = items + 12 * n
    ends = tail + 8 * (B + 1)
    _hip.call_on(index, "llj_pages_extend", slot.data_ptr(), None if add is None else add.data_ptr(), B, seen.data_ptr(), slots, table.data_ptr(), width,
                 free.data_ptr(), nfree.data_ptr(), cap, page, int(commit), tail, tail + 4 * (B + 1), rows, rows + 4 * M, rows + 8 * M, M,
                 items, n, chunk, ends, ends + 4 * B, ends + 4 * B + 4, None if fault is None else fault.data_ptr())
    return PageRows(row0, item0, row_seq, pos, place, work.view(n, 3) if chunk else None, after, left, status)


def release(table: torch.Tensor, seen: torch.Tensor, free: torch.Tensor, nfree: torch.Tensor, slot: torch.Tensor, page: int,
            fault: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The pages of these slots' sequences back onto the stack; the slots are empty behind it. Returns the status (1)."""
    index, slots, width, B, cap = _tables(table, seen, free, nfree, slot, page)
    if fault is not None and ints(fault, "fault", 1, index) != 1:
        raise ValueError("fault is one int32")
    status = table.new_empty(1)
    _hip.call_on(index, "llj_pages_release", slot.data_ptr(), B, seen.data_ptr(), slots, table.data_ptr(), width, free.data_ptr(), nfree.data_ptr(),
                 cap, page, status.data_ptr(), _hip.ptr(fault))
    return status
