"""Per-sequence state of models whose layers keep something other than a plain K / V cache.

`SequenceState` owns, for `slots` sequences at a time,
  * every recurrent layer's state (fp32, mixer.state_shape),
  * every latent-attention layer's ring of the last tokens' latents, one per layer that projects its own
    (layers that read another layer's latents have none), sized by the widest window among its readers,
  * every full-attention layer's K / V rows, the same buffers with a row for every position: as many as the
    longest sequence allowed, or without a limit as many as the longest has needed so far (`ensure`); or, with cache="int4", the
    layers' rows in 4 bits in pages that sequences take as they grow (kv4, pages: one block table for all layers),
  * the previous token of each sequence (models whose embedding looks back one token).
A sequence holds a slot from `alloc` to `release`; kernels address everything through the slot number, so
the rows of a batch need not be neighbours in memory and a batch can shrink without moving state.
"""
from __future__ import annotations

import torch

from . import kv4, pages

ALL_POSITIONS = -1  # mixer.ring_window() of layers that keep every token
GROW_ROWS = 256  # unlimited layers grow by multiples of this many rows
PAGE = 64  # tokens of a page


class SequenceState:
    def __init__(self, model, slots: int, max_length: int | None = None, cache: str | None = None):
        """max_length: no sequence will be longer (rings are capped at it); None: unbounded. cache: "int4" keeps the rows of
        full-attention layers in 4 bits (None: in the model's type)."""
        if cache not in (None, "int4"):
            raise ValueError(f"cache {cache!r}: None or 'int4'")
        self.model, self.max_length, self.cache = model, max_length, cache
        self.slots = 0
        self.recurrent: dict = {}
        self.ring: dict = {}
        self.ring_rows: dict = {}
        for i, mixer in enumerate(model.mixers):
            w = mixer.ring_window()
            if w == ALL_POSITIONS:
                self.ring_rows[i] = 0 if max_length is None else max(1, max_length)
            elif w is not None:
                self.ring_rows[i] = w if max_length is None else max(1, min(w, max_length))
        self._all = [i for i, mixer in enumerate(model.mixers) if mixer.ring_window() == ALL_POSITIONS]
        self.layout: dict = {}
        self.pool: dict = {}
        if cache is not None:
            if not self._all:
                raise ValueError("this model has no layers that keep every token: no cache to hold in 4 bits")
            for i in self._all:
                del self.ring_rows[i]
                self.layout[i] = model.mixers[i].cache_layout(PAGE)
                self.layout[i].block_bytes()  # (sizes that the cache does not take are an error here)
        self._free: list = []
        self._grow(slots)

    def _grow(self, slots: int) -> None:
        m, dev = self.model, self.model.device
        for i, mixer in enumerate(m.mixers):
            shape = mixer.state_shape()
            if shape is not None:
                self.recurrent[i] = torch.zeros(slots, *shape, dtype=torch.float32, device=dev)
            if i in self.ring_rows:
                self.ring[i] = torch.zeros(slots, self.ring_rows[i], mixer.cache_width(m.dtype), dtype=m.dtype, device=dev)
        if self.cache is not None:
            self._pages = [0] * slots  # pages kept for each sequence: of as many tokens as `room` was asked for
            width = 1 if self.max_length is None else max(1, -(-self.max_length // PAGE))
            self.table = torch.full((slots, width), -1, dtype=torch.int32, device=dev)
            self.seen = torch.zeros(slots, dtype=torch.int32, device=dev)
            self.free = torch.arange(slots, dtype=torch.int32, device=dev)
            self.nfree = torch.full((1,), slots, dtype=torch.int32, device=dev)
            self.fault = torch.zeros(1, dtype=torch.int32, device=dev)
            self.pool = {i: layout.pool(slots, dev) for i, layout in self.layout.items()}
        self.prev = torch.full((slots,), -1, dtype=torch.int32, device=dev)
        self._free = list(range(slots))
        self.slots = slots

    def room(self, slots: list, lengths: list) -> bool:
        """Room for the sequences in these slots up to so many tokens each; True if something moved (a captured step must be captured
        again)."""
        if self.cache is None:
            return self.ensure(max(lengths))
        if self.max_length is not None and max(lengths) > self.max_length:
            raise ValueError(f"sequence of {max(lengths)} tokens in a state for {self.max_length}")
        for s, n in zip(slots, lengths):
            self._pages[s] = max(self._pages[s], -(-n // PAGE))
        moved, width = False, max(self._pages)
        if width > self.table.shape[1]:
            table = torch.full((self.slots, max(width, 2 * self.table.shape[1])), -1, dtype=torch.int32, device=self.table.device)
            table[:, :self.table.shape[1]] = self.table
            self.table, moved = table, True
        have, need = self.free.numel(), sum(self._pages)
        if need > have:
            n = max(need, have + have // 2)
            free = torch.zeros(n, dtype=torch.int32, device=self.free.device)
            free[:have] = self.free
            new = torch.arange(have, n, dtype=torch.int32, device=self.free.device)
            free.index_copy_(0, (self.nfree + new - have).long(), new)  # onto the stack, whose height only the device knows
            self.free = free
            self.nfree += n - have
            for i, old in self.pool.items():
                self.pool[i] = self.layout[i].pool(n, old.device)
                self.pool[i][:have] = old
            moved = True
        return moved

    def extend(self, rows: "Rows") -> pages.PageRows:
        """Places in the pages for a call's rows (one block table for all layers), once a call. The rows go on where their sequences
        end; a prompt-style call at other positions is a fault (`check`)."""
        add = None if rows.decode else rows.new_tokens()
        out = pages.extend(self.table, self.seen, self.free, self.nfree, rows.slot, add, rows.M, PAGE, fault=self.fault)
        if not rows.decode:
            self.fault.bitwise_or_((out.pos != rows.pos).any().int() << 2)
        return out

    def ensure(self, length: int) -> bool:
        """Room for sequences of `length` tokens in the layers that keep every token; True if they moved (a captured
        step must be captured again)."""
        if not self._all or length <= self.ring_rows[self._all[0]]:
            return False
        if self.max_length is not None:
            raise ValueError(f"sequence of {length} tokens in a state for {self.max_length}")
        rows = max(-(-length // GROW_ROWS) * GROW_ROWS, 2 * self.ring_rows[self._all[0]])
        for i in self._all:
            old = self.ring[i]
            new = torch.zeros(old.shape[0], rows, old.shape[2], dtype=old.dtype, device=old.device)
            new[:, :old.shape[1]] = old
            self.ring[i], self.ring_rows[i] = new, rows
        return True

    def reserve(self, n: int) -> None:
        """Room for n more sequences; only an idle state can grow."""
        if n <= len(self._free):
            return
        if len(self._free) != self.slots:
            raise RuntimeError(f"{n} sequences asked for, {len(self._free)} of {self.slots} slots free")
        self._grow(n)

    def alloc(self, n: int) -> list:
        """n slots with the state of an empty sequence."""
        if n > len(self._free):
            raise RuntimeError(f"{n} sequences asked for, {len(self._free)} of {self.slots} slots free")
        out, self._free = self._free[:n], self._free[n:]
        idx = torch.tensor(out, dtype=torch.long, device=self.prev.device)
        for s in self.recurrent.values():
            s.index_fill_(0, idx, 0.0)
        self.prev.index_fill_(0, idx, -1)  # ring rows are only read at positions the sequence has written
        return out

    def release(self, slots) -> None:
        slots = list(slots)
        for k, s in enumerate(slots):
            if s in self._free or not 0 <= s < self.slots or s in slots[:k]:
                raise ValueError(f"slot {s} is not in use")
        if self.cache is not None:
            for k in range(0, len(slots), pages.MAX_SEQUENCES):
                ids = torch.tensor(slots[k:k + pages.MAX_SEQUENCES], dtype=torch.int32, device=self.table.device)
                pages.release(self.table, self.seen, self.free, self.nfree, ids, PAGE, self.fault)
            for s in slots:
                self._pages[s] = 0
        self._free.extend(slots)  # a freed slot is used again after every other free one

    def nbytes(self) -> int:
        own = [self.table, self.seen, self.free] if self.cache is not None else []
        return sum(t.numel() * t.element_size() for t in [*self.recurrent.values(), *self.ring.values(), *self.pool.values(), *own, self.prev])

    def check(self) -> None:
        """Waits for the calls so far and raises if one of them found no place for its rows, or had them elsewhere."""
        if self.cache is not None and int(self.fault):
            raise RuntimeError("a call's rows found no pages, or did not begin where their sequences end: this state's sequences are not valid")


class Rows:
    """The activation rows of one forward call. `decode`: one row per sequence, positions and tokens on
    the device (`pos` is advanced by the embedding). Otherwise the packed rows of every sequence's new
    tokens, sequence b's at row0[b] .. row0[b + 1] - 1 with positions start[b] ..."""

    def __init__(self, M, B, tok, pos, slot, row_seq=None, row0=None, lengths=None, starts=None):
        self.M, self.B = M, B
        self.tok, self.pos, self.slot, self.row_seq, self.row0 = tok, pos, slot, row_seq, row0
        self.lengths, self.starts = lengths, starts
        self.decode = row_seq is None
        self.slots = None  # host copy of slot (packed rows)
        self._tables: dict = {}

    @classmethod
    def packed(cls, tokens: list, starts: list, slots: list, device) -> "Rows":
        """tokens: per sequence a list of ids."""
        lengths = [len(t) for t in tokens]
        if not lengths or min(lengths) < 1:
            raise ValueError("every sequence of a call needs at least one token")
        B, M = len(lengths), sum(lengths)
        row0 = [0]
        for n in lengths:
            row0.append(row0[-1] + n)
        meta = [t for seq in tokens for t in seq]
        meta += [s + j for s, n in zip(starts, lengths) for j in range(n)]
        meta += [b for b, n in enumerate(lengths) for _ in range(n)]
        meta += row0 + list(slots)
        d = torch.tensor(meta, dtype=torch.int32).to(device)
        r = cls(M, B, d[:M], d[M:2 * M], d[3 * M + B + 1:], d[2 * M:3 * M], d[3 * M:3 * M + B + 1], lengths, list(starts))
        r.slots = list(slots)
        return r

    def _table(self, key, make):
        if key not in self._tables:
            self._tables[key] = make()
        return self._tables[key]

    def _device(self, values: list) -> torch.Tensor:
        return torch.tensor(values, dtype=torch.int32).to(self.pos.device)

    def new_tokens(self) -> torch.Tensor:
        """The sequences' numbers of rows, on the device (packed rows)."""
        return self._table("new", lambda: self._device(self.lengths))

    def chunks(self, C: int):
        """Packed rows cut into chunks of at most C tokens of one sequence: (number, table [(first row, rows,
        sequence)], each sequence's first chunk), the tables on the device."""

        def make():
            tab, first, row = [], [0], 0
            for b, n in enumerate(self.lengths):
                for j in range(0, n, C):
                    tab += [row + j, min(C, n - j), b]
                row += n
                first.append(len(tab) // 3)
            d = self._device(tab + first)
            return len(tab) // 3, d[:len(tab)], d[len(tab):]

        return self._table(("chunks", C), make)

    def pairs(self, C: int):
        """Work items of causal attention over blocks of at most C rows of one sequence: (number, table [(first row,
        rows, sequence) twice]) -- a late block, which sees many keys, with an early one (rows 0: none)."""

        def make():
            tab, row = [], 0
            for b, n in enumerate(self.lengths):
                blocks = [[row + j, min(C, n - j), b] for j in range(0, n, C)]
                row += n
                while blocks:
                    late = blocks.pop()
                    tab.append(late + (blocks.pop(0) if blocks else [0, 0, 0]))
            # the items with the most keys first
            pos = [s - r0 for s, r0 in zip(self.starts, self._row0())]
            tab.sort(key=lambda w: -(pos[w[2]] + w[0] + w[1]))
            return len(tab), self._device([x for w in tab for x in w])

        return self._table(("pairs", C), make)

    def _row0(self) -> list:
        out, row = [], 0
        for n in self.lengths:
            out.append(row)
            row += n
        return out

    def keys(self, window: int):
        """The keys the packed rows of a call may see through `window`: (number, gather or None, key0, kpos0,
        nkey), per sequence the first key row, its position and the number of rows. Without earlier tokens
        the key rows are the activation rows; otherwise gather = (source rows, -1 - nothing: from the ring;
        positions; slots) of every key row."""

        def make():
            old = [min(s, window - 1) for s in self.starts]
            key0, n = [], 0
            for o, t in zip(old, self.lengths):
                key0.append(n)
                n += o + t
            kpos0 = [s - o for s, o in zip(self.starts, old)]
            nkey = [o + t for o, t in zip(old, self.lengths)]
            B = self.B
            if not any(old):
                d = self._device(key0 + kpos0 + nkey)
                return n, None, d[:B], d[B:2 * B], d[2 * B:]
            src, kpos, kslot, row = [], [], [], 0
            for b, (o, t) in enumerate(zip(old, self.lengths)):
                src += [-1] * o + list(range(row, row + t))
                kpos += range(kpos0[b], kpos0[b] + o + t)
                kslot += [self.slots[b]] * (o + t)
                row += t
            d = self._device(key0 + kpos0 + nkey + src + kpos + kslot)
            g = d[3 * B:]
            return n, (g[:n], g[n:2 * n], g[2 * n:]), d[:B], d[B:2 * B], d[2 * B:3 * B]

        return self._table(("keys", window), make)
