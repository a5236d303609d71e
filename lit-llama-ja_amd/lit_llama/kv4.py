"""A paged K / V cache in 4 bits and grouped-query attention over it (csrc/kv4.h, kv4.hip, kv4_attend.hip).

A head's key or value is held as codes 0 .. 15 with a bf16 scale and offset, 4 + n / 2 bytes for n values (the layout and the rounding:
include/lit_llama_amd.h), so a token costs 0.27 of its bf16 bytes at heads of 128. `Layout` names the sizes, `write` puts rows where
`pages.extend` placed them, `attend` runs rows over their sequences' pages. Rows are bfloat16 or float32; scores, softmax and sums are fp32.
"""
from __future__ import annotations

from dataclasses import dataclass
from functools import lru_cache
from typing import Optional, Tuple

import torch

from . import _hip
from .pages import PAGE_SIZES, ints, on_device

# Key ranges of a call, at most. Few rows: a range is at least a round of its workgroup's waves, from 16 ranges on two (one sequence of 16,000 keys, 8
# K / V heads: 32 ranges 14.2 us, 64 18.0; of 4,000: 16 ranges 10.1, 4 12.7), and 512 workgroups or, of ranges of 1,024 keys, three on a CU (24 sequences
# of 4,000: 4 ranges 24.5 us, 2 26.4, one 29.5; 32 of 8,000: 3 ranges 49.2, one 54.6; 32 of 2,000: 2 ranges 19.3, one 18.8, 4 21.0). A sequence
# that is shorter than the table allows takes fewer by itself.
# Prompt rows: a tile of 64 keys takes TILE us, half as much again with two workgroups on a CU, 0.7 of it where there are so few that columns are
# halved (csrc/kv4_flash.hip); ranges take a launch of JOIN us that reads what they wrote at PART bytes a us, there and back, and RANGE_STEP us
# more a range. Taken is the number with the least sum, of those that fill half the CUs, all, and twice, and the root of TILE tiles / (what a range
# costs): within 13 % of the best of 12 numbers in 14 calls (512 rows behind 60,000 tokens: 4 ranges 681 us, one 1,445; 128 rows of 8 heads' keys
# behind 2,048: 4 ranges 24, 16 33, one 55; 24 rows of 20 fp32 heads on one behind 9,400: 31 ranges 33, 10 47; 512 rows of a prompt alone: one
# 19.4, two 28.8).
WGS, WGS_LONG = 512, 768
RANGE, RANGES, RANGE_LONG = 256, 16, 1024
TILE, JOIN, RANGE_STEP, PART = 2.2, 4.0, 0.2, 4e6
FEW_COLUMNS = 64  # (row, head) pairs of a K / V head in an item: from more on it is prompt rows (csrc/kv4_attend.hip)


# (sizes, functions of a few integers: asked of the library once each, a call into it takes five times as long)
@lru_cache(None)
def _block_bytes(page: int, dim: int, vdim: int) -> int:
    return int(_hip.lib().llj_kv4_block_bytes(page, dim, vdim))


@lru_cache(4096)
def _tiles(heads: int, kv_heads: int, dim: int, vdim: int, rows: int, dt: int) -> int:
    return int(_hip.lib().llj_kv4_tiles(heads, kv_heads, dim, vdim, rows, dt))


@lru_cache(None)
def _part_bytes(vdim: int) -> int:
    return 4 * int(_hip.lib().llj_kv4_part_width(vdim))


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
        n = _block_bytes(self.page, self.dim, self.vdim)
        if n == 0 or self.kv_heads < 1:
            raise ValueError(f"{self}: pages of {PAGE_SIZES} tokens, heads of 1 to 256")
        return n

    def pool(self, pages: int, device="cuda") -> torch.Tensor:
        """A cache of this many pages, every place zero."""
        return torch.zeros(pages, self.kv_heads, self.block_bytes(), dtype=torch.uint8, device=device)


def _pool(pool: torch.Tensor, layout: Layout) -> tuple:
    """(device, pages)"""
    if not isinstance(pool, torch.Tensor) or pool.dtype != torch.uint8 or pool.dim() != 3 or not pool.is_contiguous():
        raise ValueError("pool must be a contiguous uint8 tensor (pages, kv_heads, bytes)")
    pages, G, n = pool.shape
    if G != layout.kv_heads or n != layout.block_bytes() or not pages:
        raise ValueError(f"pool {tuple(pool.shape)} does not fit {layout}")
    if pages * layout.page > 1 << 30:
        raise ValueError(f"{pages} pages of {layout.page} tokens: up to 2^30 tokens are taken")
    return on_device(pool, "pool"), pages


def _heads(t: torch.Tensor, what: str, M: int, heads: int, n: int, index: int) -> Tuple[int, int]:
    """(row stride, head stride) of rows (M, heads, n) or (M, heads n)."""
    if on_device(t, what) != index:
        raise ValueError(f"{what} is on {t.device}, the cache on cuda:{index}")
    st = t.stride()
    if t.shape == (M, heads, n) and (n == 1 or st[2] == 1):
        ld, hs = st[0], st[1]
    elif t.shape == (M, heads * n) and (heads * n == 1 or st[1] == 1):
        ld, hs = st[0], n
    else:
        raise ValueError(f"{what} {tuple(t.shape)}: ({M}, {heads}, {n}) or ({M}, {heads * n}) with a head's values one after another")
    if ld >> 40 or hs >> 40:
        raise ValueError(f"{what}: strides {st}")
    return ld, hs


def _lead(t: torch.Tensor, what: str, M: int, n: int, index: int) -> int:
    """Row stride of rows (M, n) whose values follow one another."""
    if t.dim() != 2 or t.shape != (M, n):
        raise ValueError(f"{what} {tuple(t.shape)}: ({M}, {n})")
    return _stride(t, what, M, n, index)


def _stride(t: torch.Tensor, what: str, M: int, n: int, index: int) -> int:
    if t.get_device() != index:
        raise ValueError(f"{what} is on {t.device}, the cache on cuda:{index}")
    ld, one = t.stride()
    if M == 1:
        ld = n
    if (one != 1 and n > 1) or not n <= ld < 1 << 31:
        raise ValueError(f"{what}: rows of {n} with strides {t.stride()}")
    return ld


def write(pool: torch.Tensor, layout: Layout, k: torch.Tensor, v: torch.Tensor, place: torch.Tensor) -> None:
    """Keys (M, kv_heads, dim) and values (M, kv_heads, vdim) into place[m] (< 0: the row is left out). The places of a call differ."""
    index, pages = _pool(pool, layout)
    M = ints(place, "place", 1, index)
    if k.dtype != v.dtype:
        raise TypeError(f"keys are {k.dtype}, values {v.dtype}")
    G, D, V = layout.kv_heads, layout.dim, layout.vdim
    ldk, hk = _heads(k, "k", M, G, D, index)
    ldv, hv = _heads(v, "v", M, G, V, index)
    _hip.call_on(index, "llj_kv4_write", k.data_ptr(), ldk, hk, v.data_ptr(), ldv, hv, place.data_ptr(), M, G, D, V, _dt(k.dtype), pool.data_ptr(),
                 pages, layout.page)


def read(pool: torch.Tensor, layout: Layout, place: torch.Tensor, dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
    """What stands at place[m]: keys (M, kv_heads, dim) and values (M, kv_heads, vdim); zeros for a place outside the pool."""
    index, pages = _pool(pool, layout)
    M, dt = ints(place, "place", 1, index), _dt(dtype)
    G, D, V = layout.kv_heads, layout.dim, layout.vdim
    k = pool.new_empty(M, G, D, dtype=dtype)
    v = pool.new_empty(M, G, V, dtype=dtype)
    _hip.call_on(index, "llj_kv4_read", pool.data_ptr(), pages, layout.page, place.data_ptr(), M, G, D, V, dt, k.data_ptr(), G * D, D, v.data_ptr(),
                 G * V, V)
    return k, v


def splits(layout: Layout, heads: int, items: int, rows: int, keys: int, dtype: torch.dtype = torch.bfloat16) -> Tuple[int, int]:
    """(key ranges, counters) of a call of `items` items of up to `rows` rows over up to `keys` keys (prompt rows need no counters)."""
    tiles = _tiles(heads, layout.kv_heads, layout.dim, layout.vdim, rows, _dt(dtype))
    if not tiles:
        raise ValueError(f"{heads} heads on {layout.kv_heads}, items of {rows} rows")
    wgs = max(1, items * tiles)
    if rows * heads // layout.kv_heads > FEW_COLUMNS:
        return _prompt_splits(wgs, -(-keys // 64), rows * heads / tiles * _part_bytes(layout.vdim) * 2 / PART), 0
    if keys <= (2 if max(layout.dim, layout.vdim) <= 128 else 1) * RANGE:  # (two rounds of four waves: the device makes one range of it)
        return 1, items * tiles
    long = -(-keys // RANGE_LONG)
    n = -(-keys // RANGE)
    if n > RANGES:
        n = max(RANGES, -(-keys // (2 * RANGE)))
    return max(1, min(64, max(min(n, WGS // wgs), min(long, WGS_LONG // wgs)))), items * tiles


@lru_cache(4096)
def _prompt_splits(wgs: int, tiles: int, part: float) -> int:
    """Key ranges of wgs workgroups over so many tiles, whose parts take `part` us a range."""
    most, each = min(64, tiles, WGS // wgs), RANGE_STEP + wgs * part
    if most < 2:
        return 1

    def us(n):
        share = 0.7 if 2 * wgs * n <= 256 else 1.0 if wgs * n <= 256 else 1.5
        return TILE * share * -(-tiles // n) + (JOIN + each * n if n > 1 else 0.0)

    tried = {1, most, *(max(1, min(most, n)) for n in (round((TILE * tiles / each) ** 0.5), 128 // wgs, 256 // wgs))}
    return min(sorted(tried), key=us)


def item_rows(layout: Layout, heads: int, longest: int) -> int:
    """Rows of a work item for sequences of up to `longest` rows in a call: few rows share the 16 columns of a tile, prompt rows the
    128 that a tile of keys is unpacked for (fp32 rows and heads over 128 in two tiles of 64; items of 64, which are few rows, took 713 us
    for 394 at 4,096 fp32 rows of 32 heads on 8)."""
    R = heads // layout.kv_heads
    return max(1, (16 if longest * R <= FEW_COLUMNS else 128) // R)


def attend(q: torch.Tensor, pool: torch.Tensor, layout: Layout, table: torch.Tensor, slot: torch.Tensor, pos: torch.Tensor, *,
           work: Optional[torch.Tensor] = None, rows: int = 1, scale: Optional[float] = None, sink: bool = False,
           gate: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, count: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Softmax attention of rows q (M, heads dim) over the positions up to pos[m] of their sequences: y (M, heads vdim).

    work: items (first row, rows, sequence) of at most `rows` rows (pages.extend's with chunk = rows); rows of no item are left as they are
    in `out`. None: row m is sequence m's. Sequence b is in table[slot[b]]. scale: dim^-0.5 by default; sink: a key of score 0 without a
    value; gate (M, heads): head h's output times sigmoid(gate[:, h]). A row with pos < 0 is zero. Rows of few keys and items are split over
    key ranges, whose counters `count` a program may keep for all its calls on one stream (int32, zero, `splits` says how many)."""
    index, pages = _pool(pool, layout)
    G, D, V, page = layout.kv_heads, layout.dim, layout.vdim, layout.page
    if q.dim() != 2 or not q.numel() or q.size(1) % (G * D):
        raise ValueError(f"q {tuple(q.shape)}: (M, heads {D}) with heads a multiple of {G}")
    M, n = q.shape
    H, dtype = n // D, q.dtype
    dt, ldq = _dt(dtype), _stride(q, "q", M, n, index)
    ints(table, "table", 2, index)
    slots, width = table.shape
    B = ints(slot, "slot", 1, index)
    if ints(pos, "pos", 1, index) != M:
        raise ValueError(f"{pos.numel()} positions for {M} rows")
    if work is None:
        items, rows, work_at = M, 1, None
        if B < M:
            raise ValueError(f"{M} rows of {B} sequences without work items")
    else:
        items, work_at = ints(work, "work", 2, index) // 3, work.data_ptr()
        if work.size(1) != 3 or rows < 1:
            raise ValueError("work items are (first row, rows, sequence), of at least one row")
    if out is None:
        out = q.new_empty(M, H * V)
        ldo = H * V
    else:
        ldo = _lead(out, "out", M, H * V, index)
    gate_at, ldg = (None, 0) if gate is None else (gate.data_ptr(), _lead(gate, "gate", M, H, index))
    if out.dtype != dtype or (gate is not None and gate.dtype != dtype):
        raise TypeError(f"q, gate and out are of one type, {dtype}")
    n, need = splits(layout, H, items, rows, width * page, dtype)
    part_at = counters = None
    if n > 1:
        part = pool.new_empty(M * H * n * _part_bytes(V))
        part_at = part.data_ptr()
        if need:
            if count is None:
                count = torch.zeros(need, dtype=torch.int32, device=q.device)
            elif ints(count, "count", 1, index) < need:
                raise ValueError(f"{count.numel()} counters, {need} are needed")
            counters = count.data_ptr()
    _hip.call_on(index, "llj_kv4_attend", q.data_ptr(), ldq, gate_at, ldg, work_at, items, rows, pos.data_ptr(), slot.data_ptr(), B, table.data_ptr(),
                 slots, width, pool.data_ptr(), pages, page, part_at, counters, n, out.data_ptr(), ldo, M, H, G, D, V,
                 D ** -0.5 if scale is None else scale, int(sink), dt)
    return out
