"""The paged 4-bit K / V cache in plain numpy, double precision: block tables, the vectors' codes, attention (test-only)."""
import numpy as np


def bf16_bits(x):
    """Bits of the bf16 nearest to float32 x (halves to even)."""
    u = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint32)


def from_bits(b):
    return (np.asarray(b, np.uint32) << 16).view(np.float32).astype(np.float64)


def floor_bits(x):
    """Bits of the largest bf16 up to float32 x."""
    u = np.asarray(x, np.float32).view(np.uint32)
    return (u >> 16) + ((u >> 31 == 1) & (u & 0xFFFF != 0)).astype(np.uint32)


def quantize(x):
    """(codes, scale, offset) of vectors x (.., n), float32 values; scale and offset NaN where a vector is not finite."""
    x = np.asarray(x, np.float32)
    good = np.isfinite(x).all(-1)
    y = np.where(good[..., None], x, 0.0).astype(np.float32)
    ob = floor_bits(y.min(-1))
    good &= (ob & 0x7F80) != 0x7F80
    o = np.where(good, from_bits(ob), 0.0)
    y = np.where(good[..., None], y, 0.0)
    s = from_bits(bf16_bits(((y.max(-1).astype(np.float64) - o) / 15.0).astype(np.float32)))
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where((s > 0)[..., None], np.clip(np.rint((y - o[..., None]) / s[..., None]), 0, 15), 0.0)
    return c, np.where(good, s, np.nan), np.where(good, o, np.nan)


def stands_for(x):
    c, s, o = quantize(x)
    return c * s[..., None] + o[..., None]


def width(n):
    return 64 if n <= 64 else 128 if n <= 128 else 256


def pack(k, v, page):
    """A page's block of one head from up to `page` keys (t, dim) and values (t, vdim): its bytes."""
    out = []
    for x in (k, v):
        c = np.zeros((page, width(x.shape[1])), np.uint8)
        c[:x.shape[0], :x.shape[1]] = quantize(x)[0]
        out.append((c[:, 0::2] | c[:, 1::2] << 4).reshape(-1))
    for x in (k, v):
        _, s, o = quantize(x)
        w = np.zeros(page, np.uint32)
        w[:x.shape[0]] = np.where(np.isnan(s), 0x7FC07FC0, bf16_bits(s.astype(np.float32)) | bf16_bits(o.astype(np.float32)) << 16)
        out.append(w.view(np.uint8))
    return np.concatenate(out)


def attend(q, k, v, pos, scale, sink=False, gate=None):
    """Rows q (M, H, D) over one sequence's keys k (L, G, D), values v (L, G, V); row m sees positions up to pos[m]."""
    M, H, _ = q.shape
    R = H // k.shape[1]
    y = np.zeros((M, H, v.shape[2]))
    for m in range(M):
        n = min(int(pos[m]) + 1, len(k))
        if n <= 0:
            continue
        for h in range(H):
            s = k[:n, h // R] @ q[m, h] * scale
            top = max(s.max(), 0.0) if sink else s.max()
            e = np.exp(s - top)
            y[m, h] = e @ v[:n, h // R] / (e.sum() + (np.exp(-top) if sink else 0.0))
        if gate is not None:
            y[m] /= (1.0 + np.exp(-gate[m]))[:, None]
    return y


class Tables:
    """Block tables kept on the host, request by request."""

    def __init__(self, table, seen, free, page):
        self.table, self.seen, self.free, self.page = [list(r) for r in table], list(seen), list(free), page

    def extend(self, slots, adds, chunk=0):
        """(row0, row_seq, pos, place, work)"""
        row0, seq, pos, place, work = [0], [], [], [], []
        for b, (x, n) in enumerate(zip(slots, adds)):
            if chunk:
                work += [[len(pos) + j, min(chunk, n - j), b] for j in range(0, n, chunk)]
            held = -(-self.seen[x] // self.page)
            for t in range(self.seen[x], self.seen[x] + n):
                if t // self.page >= held:
                    self.table[x][held] = self.free.pop()
                    held += 1
                seq.append(b)
                pos.append(t)
                place.append(self.table[x][t // self.page] * self.page + t % self.page)
            self.seen[x] += n
            row0.append(len(pos))
        return row0, seq, pos, place, work

    def release(self, slots):
        for x in slots:
            for i in range(-(-self.seen[x] // self.page)):
                self.free.append(self.table[x][i])
                self.table[x][i] = -1
            self.seen[x] = 0
