"""A paged K / V cache in 4 bits and grouped-query attention over it (csrc/kv4.h, kv4.hip, kv4_attend.hip).

A head's key or value is held as codes 0 .. 15 with a bf16 scale and offset, 4 + n / 2 bytes for n values (the layout and the rounding:
include/lit_llama_amd.h), so a token costs 0.27 of its bf16 bytes at heads of 128. `Layout` names the sizes, `write` puts rows where
`pages.extend` placed them, `attend` runs rows over their sequences' pages. Rows are bfloat16 or float32; scores, softmax and sums are fp32.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _hip
from .pages import PAGE_SIZES, _ints

WGS = 512  # workgroups that the keys of a call are split for
RANGE = 256  # the shortest key range


def _dt(t: torch.dtype) -> int:
    if t not in (torch.bfloat16, torch.float32):
        raise TypeError(f"rows are bfloat16 or float32, not {t}")
    return 0 if t == torch.bfloat16 else 1


@dataclass(frozen=True)
class Layout:
    kv_heads: int
    dim: int
    vdim: int
    page: int

    def block_bytes(self) -> int:
        """Bytes of one head's part of a page."""
        n = int(_hip.lib().llj_kv4_block_bytes(self.page, self.dim, self.vdim))
        if n == 0 or self.kv_heads < 1:
            raise ValueError(f"{self}: pages of {PAGE_SIZES} tokens, heads of 1 to 256")
        return n

    def pool(self, pages: int, device="cuda") -> torch.Tensor:
        """A cache of this many pages, every place zero."""
        return torch.zeros(pages, self.kv_heads, self.block_bytes(), dtype=torch.uint8, device=device)


def _pool(pool: torch.Tensor, layout: Layout) -> torch.device:
    if not isinstance(pool, torch.Tensor) or pool.dtype != torch.uint8 or pool.dim() != 3 or not pool.is_contiguous():
        raise ValueError("pool must be a contiguous uint8 tensor (pages, kv_heads, bytes)")
    if pool.shape[1] != layout.kv_heads or pool.shape[2] != layout.block_bytes() or not pool.shape[0]:
        raise ValueError(f"pool {tuple(pool.shape)} does not fit {layout}")
    if pool.shape[0] * layout.page > 1 << 30:
        raise ValueError(f"{pool.shape[0]} pages of {layout.page} tokens: up to 2^30 tokens are taken")
    _hip.require_device(pool, "pool")
    return pool.device


def _heads(t: torch.Tensor, what: str, M: int, heads: int, n: int, device) -> Tuple[int, int]:
    """(row stride, head stride) of rows (M, heads, n) or (M, heads n)."""
    if t.device != device:
        raise ValueError(f"{what} is on {t.device}, the cache on {device}")
    if t.dim() == 3 and tuple(t.shape) == (M, heads, n) and (n == 1 or t.stride(2) == 1):
        ld, hs = t.stride(0), t.stride(1)
    elif t.dim() == 2 and tuple(t.shape) == (M, heads * n) and (heads * n == 1 or t.stride(1) == 1):
        ld, hs = t.stride(0), n
    else:
        raise ValueError(f"{what} {tuple(t.shape)}: ({M}, {heads}, {n}) or ({M}, {heads * n}) with a head's values one after another")
    if ld >> 40 or hs >> 40:
        raise ValueError(f"{what}: strides {t.stride()}")
    return ld, hs


def _lead(t: torch.Tensor, what: str) -> int:
    """Row stride of rows (M, n)."""
    ld = t.stride(0) if t.shape[0] > 1 else t.shape[1]
    if not t.shape[1] <= ld < 1 << 31:
        raise ValueError(f"{what}: rows of {t.shape[1]} with stride {ld}")
    return ld


def write(pool: torch.Tensor, layout: Layout, k: torch.Tensor, v: torch.Tensor, place: torch.Tensor) -> None:
    """Keys (M, kv_heads, dim) and values (M, kv_heads, vdim) into place[m] (< 0: the row is left out). The places of a call differ."""
    dev = _pool(pool, layout)
    M = place.numel() if isinstance(place, torch.Tensor) else 0
    if not M:
        raise ValueError("write takes at least one row")
    _ints(place, "place", 1, dev)
    if k.dtype != v.dtype:
        raise TypeError(f"keys are {k.dtype}, values {v.dtype}")
    ks, vs = _heads(k, "k", M, layout.kv_heads, layout.dim, dev), _heads(v, "v", M, layout.kv_heads, layout.vdim, dev)
    _hip.call_on(pool, "llj_kv4_write", k.data_ptr(), *ks, v.data_ptr(), *vs, place.data_ptr(), M, layout.kv_heads, layout.dim, layout.vdim,
                 _dt(k.dtype), pool.data_ptr(), pool.shape[0], layout.page)


def read(pool: torch.Tensor, layout: Layout, place: torch.Tensor, dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
    """What stands at place[m]: keys (M, kv_heads, dim) and values (M, kv_heads, vdim); zeros for a place outside the pool."""
    dev = _pool(pool, layout)
    _ints(place, "place", 1, dev)
    M, G, dt = place.numel(), layout.kv_heads, _dt(dtype)
    k = torch.empty(M, G, layout.dim, dtype=dtype, device=dev)
    v = torch.empty(M, G, layout.vdim, dtype=dtype, device=dev)
    _hip.call_on(pool, "llj_kv4_read", pool.data_ptr(), pool.shape[0], layout.page, place.data_ptr(), M, G, layout.dim, layout.vdim, dt, k.data_ptr(),
                 G * layout.dim, layout.dim, v.data_ptr(), G * layout.vdim, layout.vdim)
    return k, v


def splits(layout: Layout, heads: int, items: int, rows: int, keys: int) -> Tuple[int, int]:
    """(key ranges, counters) of a call of `items` items of up to `rows` rows over up to `keys` keys."""
    tiles = int(_hip.lib().llj_kv4_tiles(heads, layout.kv_heads, rows))
    if not tiles:
        raise ValueError(f"{heads} heads on {layout.kv_heads}, items of {rows} rows")
    return max(1, min(64, -(-keys // RANGE), WGS // max(1, items * tiles))), items * tiles


def attend(q: torch.Tensor, pool: torch.Tensor, layout: Layout, table: torch.Tensor, slot: torch.Tensor, pos: torch.Tensor, *,
           work: Optional[torch.Tensor] = None, rows: int = 1, scale: Optional[float] = None, sink: bool = False,
           gate: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, count: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Softmax attention of rows q (M, heads dim) over the positions up to pos[m] of their sequences: y (M, heads vdim).

    work: items (first row, rows, sequence) of at most `rows` rows (pages.extend's with chunk = rows); rows of no item are left as they are
    in `out`. None: row m is sequence m's. Sequence b is in table[slot[b]]. scale: dim^-0.5 by default; sink: a key of score 0 without a
    value; gate (M, heads): head h's output times sigmoid(gate[:, h]). A row with pos < 0 is zero. Rows of few keys and items are split over
    key ranges, whose counters `count` a program may keep for all its calls on one stream (int32, zero, `splits` says how many)."""
    dev = _pool(pool, layout)
    G, D, V = layout.kv_heads, layout.dim, layout.vdim
    if q.dim() != 2 or q.shape[1] % (G * D) or not q.numel() or (q.shape[1] > 1 and q.stride(1) != 1) or q.device != dev:
        raise ValueError(f"q {tuple(q.shape)}: (M, heads {D}) with heads a multiple of {G}, on {dev}")
    M, H = q.shape[0], q.shape[1] // D
    _ints(table, "table", 2, dev)
    _ints(slot, "slot", 1, dev)
    if _ints(pos, "pos", 1, dev).numel() != M:
        raise ValueError(f"{pos.numel()} positions for {M} rows")
    if work is None:
        items, rows = M, 1
        if slot.numel() < M:
            raise ValueError(f"{M} rows of {slot.numel()} sequences without work items")
    elif _ints(work, "work", 2, dev).shape[1] != 3 or rows < 1:
        raise ValueError("work items are (first row, rows, sequence), of at least one row")
    else:
        items = work.shape[0]
    dt = _dt(q.dtype)
    if gate is not None and (tuple(gate.shape) != (M, H) or gate.dtype != q.dtype or (H > 1 and gate.stride(1) != 1) or gate.device != dev):
        raise ValueError(f"gate must be ({M}, {H}) of {q.dtype}")
    if out is None:
        out = torch.empty(M, H * V, dtype=q.dtype, device=dev)
    elif tuple(out.shape) != (M, H * V) or out.dtype != q.dtype or (H * V > 1 and out.stride(1) != 1) or out.device != dev:
        raise ValueError(f"out must be ({M}, {H * V}) of {q.dtype}")
    n, need = splits(layout, H, items, rows, table.shape[1] * layout.page)
    part = None
    if n > 1:
        part = torch.empty(M * H * n * _hip.lib().llj_kv4_part_width(V), dtype=torch.float32, device=dev)
        if count is None:
            count = torch.zeros(need, dtype=torch.int32, device=dev)
        elif _ints(count, "count", 1, dev).numel() < need:
            raise ValueError(f"{count.numel()} counters, {need} are needed")
    _hip.call_on(pool, "llj_kv4_attend", q.data_ptr(), _lead(q, "q"), _hip.ptr(gate), 0 if gate is None else _lead(gate, "gate"), _hip.ptr(work), items, rows,
                 pos.data_ptr(), slot.data_ptr(), slot.numel(), table.data_ptr(), table.shape[0], table.shape[1], pool.data_ptr(), pool.shape[0],
                 layout.page, _hip.ptr(part), _hip.ptr(count) if n > 1 else None, n, out.data_ptr(), _lead(out, "out"), M, H, G, D, V,
                 D ** -0.5 if scale is None else scale, int(sink), dt)
    return out
