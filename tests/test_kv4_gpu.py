"""The paged 4-bit K / V cache (csrc/kv4.hip, kv4_attend.hip) against oracle/kv4_np.py in double precision.

Codes, scales and offsets are compared bit for bit. Attention's tolerance, for rows y = sum_j p_j v_j (derived, not fitted):
  * the output's rounding, eps / 2 of its type, relative to |y|; the gate's sigmoid some fp32 roundings, 2^-21;
  * a score is a sum of D products of bf16 numbers with 16 + c <= 31, accumulated in fp32, scaled, plus offset times the queries' sum:
    |error| <= e = (D + 8) 2^-24 scale (31 s + |o|) sum |q| at most, the queries themselves exact (three bf16 terms);
    every weight is then off by a factor exp(2 e) at most (its own score and the sum's), and by 2^-21 from exp2, whose argument is rounded: 2^-23
    |score - top|, both times max |v|;
  * a weight times its scale enters as one fp16 number or as two, and is summed over n keys in fp32, n 2^-24, beside 16 + c: times (31 s + |o|) of
    the values. Of two numbers (22 bits) 2^-24 is allowed. Of one, each off by up to 2^-11 p (15 s) and
    of either sign, the bf16 output's own 2^-8 |y| covers it where |y| is of the values' size; 2^-16 is allowed beside it where it is not.
"""
import numpy as np
import pytest
import torch

from oracle import kv4_np as O

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float32]


def ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32).cuda()


def rounded(a, dtype):
    """Values of the type, as numpy float64 and on the device."""
    t = torch.tensor(np.asarray(a), dtype=torch.float32).to(dtype)
    return t.double().numpy(), t.cuda()


def keys(g, *shape):
    """Channels of different spread around means of their own, a few of them large."""
    mean = g.standard_normal(shape[1:]) * (1 + 6 * (g.random(shape[1:]) < 0.04))
    return g.standard_normal(shape) * g.uniform(0.5, 1.5, shape[1:]) + mean


def same(a, b):
    return np.array_equal(a, b, equal_nan=True)


# ------------------------------------------------------------------------------------------- rows in and out
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,G,D,V,page", [(1, 1, 64, 64, 16), (5, 2, 128, 128, 64), (33, 3, 78, 78, 16), (70, 2, 1, 3, 32), (19, 1, 256, 200, 128),
                                          (300, 4, 96, 64, 256), (9, 2, 65, 129, 64), (40, 10, 64, 64, 16), (7, 1, 128, 250, 16), (1003, 5, 24, 8, 32)])
def test_rows_in_and_out(hip, dtype, M, G, D, V, page):
    """The bytes of every page, and what is read back in both types; the pages between are left as they were."""
    from lit_llama import kv4

    g = np.random.default_rng(M + D)
    lay = kv4.Layout(G, D, V, page)
    n = -(-M // page) + 2
    pool = lay.pool(n)
    pool.fill_(0xA5)
    k, kd = rounded(keys(g, M, G, D), dtype)
    v, vd = rounded(g.standard_normal((M, G, V)), dtype)
    place = g.permutation(n * page)[:M]
    kv4.write(pool, lay, kd, vd, ints(place))
    want = np.full((n, G, lay.block_bytes()), 0xA5, np.uint8)
    kb, vb = O.width(D) // 2, O.width(V) // 2
    for m, at in enumerate(place):
        p, t = divmod(int(at), page)
        for h in range(G):
            b = O.pack(k[m, h][None], v[m, h][None], page)
            c, s = page * kb, page * (kb + vb)
            for base, size in ((0, kb), (c, vb), (s, 4), (s + 4 * page, 4)):
                want[p, h, base + t * size:base + (t + 1) * size] = b[base:base + size]
    assert np.array_equal(pool.cpu().numpy(), want)
    for out in DTYPES:
        a, b = kv4.read(pool, lay, ints(place), out)
        assert same(a.double().cpu().numpy(), rounded(O.stands_for(k), out)[0])
        assert same(b.double().cpu().numpy(), rounded(O.stands_for(v), out)[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_vectors_on_the_edges(hip, dtype):
    """Constant vectors, values on the border between two codes, zeros of both signs, subnormal spreads, the type's largest values, a large
    common part, infinities and NaN in one vector beside good ones."""
    from lit_llama import kv4

    D, G = 64, 1
    top = float(torch.finfo(dtype).max)
    g = np.random.default_rng(3)
    x = np.zeros((14, G, D))
    x[1] = 1.375
    x[2] = -0.0
    x[3, 0] = np.linspace(-7.5, 7.5, D)  # (o = -7.5, s = 1: every half is a border)
    x[3, 0, ::4] = 0.0
    x[4, 0] = np.arange(D) % 31 * 0.5
    x[5, 0, ::2], x[5, 0, 1] = top, -3.3e38
    x[6, 0, 3] = 1e-39
    x[7, 0] = 1000 + g.standard_normal(D)
    x[8, 0, 5] = np.inf
    x[9, 0, 5] = -np.inf
    x[10, 0, 5] = np.nan
    x[11, 0] = g.standard_normal(D) * 1e-30
    x[12, 0] = -top
    x[13, 0] = np.where(np.arange(D) % 2, 1e-30, -1.0)
    k, kd = rounded(x, dtype)
    lay = kv4.Layout(G, D, D, 16)
    pool = lay.pool(1)
    kv4.write(pool, lay, kd, kd, ints(np.arange(14)))
    a, b = kv4.read(pool, lay, ints(np.arange(14)))
    with np.errstate(over="ignore"):  # (code 15 of the widest vector stands for more than a float32 holds)
        want = O.stands_for(k).astype(np.float32).astype(np.float64)
    assert same(a.double().cpu().numpy(), want) and same(b.double().cpu().numpy(), want)
    assert np.isnan(want[8:11]).all() and np.isfinite(O.stands_for(k)[:8]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_places_outside(hip, dtype):
    """Rows out of packed projections at odd columns, heads with gaps, rows whose place is -1 or behind the pool."""
    from lit_llama import kv4

    g = np.random.default_rng(5)
    M, G, D, V = 21, 3, 40, 24
    lay = kv4.Layout(G, D, V, 16)
    wide, wd = rounded(keys(g, M, G * (D + V) + 7), dtype)
    k, v = wd[:, 3:3 + G * D], wd[:, 3 + G * D:3 + G * (D + V)]
    place = np.arange(M) + 5
    place[4], place[9], place[15] = -1, 48, 1 << 30
    pool = lay.pool(3)
    pool.fill_(0x5A)
    kv4.write(pool, lay, k, v, ints(place))
    a, b = kv4.read(pool, lay, ints(place))
    good = np.array([0 <= p < 48 for p in place])
    wk = O.stands_for(wide[:, 3:3 + G * D].reshape(M, G, D))
    wv = O.stands_for(wide[:, 3 + G * D:3 + G * (D + V)].reshape(M, G, V))
    assert same(a.double().cpu().numpy()[good], wk[good].astype(np.float32)) and same(b.double().cpu().numpy()[good], wv[good].astype(np.float32))
    assert not a[torch.tensor(~good).cuda()].any() and not b[torch.tensor(~good).cuda()].any()
    used = set(place[good])
    left, _ = kv4.read(pool, lay, ints([p for p in range(48) if p not in used]))
    assert torch.equal(left, left[:1, :1].expand_as(left))  # (the filling, everywhere else)
    # heads with gaps between them
    gaps, gd = rounded(keys(g, M, G, D + V + 1), dtype)
    kv4.write(pool, lay, gd[:, :, 1:1 + D], gd[:, :, 1 + D:], ints(np.arange(M)))
    a, b = kv4.read(pool, lay, ints(np.arange(M)))
    assert same(a.double().cpu().numpy(), O.stands_for(gaps[:, :, 1:1 + D]).astype(np.float32))
    assert same(b.double().cpu().numpy(), O.stands_for(gaps[:, :, 1 + D:]).astype(np.float32))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,G,D,V,RD,norm,mix", [(4, 2, 64, 64, 64, 1, None), (8, 2, 128, 128, 32, 1, "copy"), (6, 3, 78, 78, 10, 0, "mix"), (5, 1, 40, 200, 0, 1, "mix"),
                                                 (3, 3, 256, 130, 256, 1, None), (4, 4, 33, 17, 2, 1, "copy"), (40, 10, 64, 64, 64, 1, "mix"), (2, 1, 8, 1, 8, 0, None),
                                                 (64, 64, 256, 256, 64, 1, None), (96, 96, 256, 256, 64, 1, None)])
def test_prepared_rows(hip, dtype, H, G, D, V, RD, norm, mix):
    """llj_gqa_prep_kv4: the pool's bytes, the queries and the values kept aside are those of llj_gqa_prep into plain rows and write out of them. Rows
    without a place prepare their queries all the same. 96 fp32 heads of 256 + 256 (192 KiB a row) are refused."""
    from lit_llama import _hip, kv4

    g = np.random.default_rng(H + D)
    M, page = 19, 32
    oq, ok, ov, ld = 8, 8 + H * D, 16 + (H + G) * D, 24 + (H + G) * D + G * V
    ld += -ld % 8
    _, x = rounded(g.standard_normal((M, ld)), dtype)
    _, f0 = rounded(g.standard_normal((M, G * V + 3)), dtype)
    lam = torch.tensor([0.3], device="cuda")
    turns = torch.tensor(g.random(max(RD // 2, 1)), dtype=torch.float64, device="cuda")
    pos, slot = ints(g.integers(0, 64, M)), ints(range(M))
    place = g.permutation(5 * page)[:M]
    place[4], place[11] = -1, 5 * page
    place, lay, dt = ints(place), kv4.Layout(G, D, V, page), 0 if dtype == torch.bfloat16 else 1
    out = []
    for fused in (False, True):
        y, f, pool = x.clone(), f0.clone(), lay.pool(5)
        head = (y.data_ptr(), ld, oq, ok, ov, turns.data_ptr(), RD, norm, 1e-5)
        keep = (f.data_ptr() if mix else None, lam.data_ptr() if mix == "mix" else None, f.stride(0))
        tail = (M, H, G, D, V, dt, _hip.stream())
        if fused:
            args = (*head, pos.data_ptr(), place.data_ptr(), pool.data_ptr(), 5, page, *keep, *tail)
            if G * (D + V) * dtype.itemsize > 160 * 1024 - 4 * RD:
                with pytest.raises(_hip.HipError):
                    _hip.call("llj_gqa_prep_kv4", *args)
                return
            _hip.call("llj_gqa_prep_kv4", *args)
        else:
            ldc = -(-G * (D + V) // 8) * 8
            cache = torch.empty(M, 64, ldc, dtype=dtype, device="cuda")
            _hip.call("llj_gqa_prep", *head, pos.data_ptr(), None, slot.data_ptr(), cache.data_ptr(), 64, ldc, *keep, *tail)
            kv = cache[torch.arange(M, device="cuda"), pos.long()]
            kv4.write(pool, lay, kv[:, :G * D], kv[:, G * D:G * (D + V)], place)
        out.append((y, f, pool))
    for a, b in zip(*out):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("G,D,V", [(64, 256, 256), (7, 64, 96), (16, 130, 20)])
def test_prepared_rows_in_one_workgroup_each(hip, dtype, G, D, V):
    """520 rows of a call, whose heads stay in one workgroup (128 KiB of keys and values in fp32), against calls of 8 rows, whose heads are spread."""
    from lit_llama import _hip, kv4

    g = np.random.default_rng(G)
    M, page, H = 520, 64, 2 * G
    ld = (H + G) * D + G * V
    _, x = rounded(g.standard_normal((M, ld)), dtype)
    turns = torch.tensor(g.random(16), dtype=torch.float64, device="cuda")
    pos, place, lay, dt = ints(range(M)), ints(g.permutation(9 * page)[:M]), kv4.Layout(G, D, V, page), 0 if dtype == torch.bfloat16 else 1
    out = []
    for n in (520, 8):
        y, pool = x.clone(), lay.pool(9)
        for m in range(0, M, n):
            _hip.call("llj_gqa_prep_kv4", y[m:].data_ptr(), ld, 0, H * D, (H + G) * D, turns.data_ptr(), 32, 1, 1e-5, pos[m:].data_ptr(), place[m:].data_ptr(),
                      pool.data_ptr(), 9, page, None, None, 0, n, H, G, D, V, dt, _hip.stream())
        out.append((y, pool))
    for a, b in zip(*out):
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------- attention
class Case:
    """Sequences of `lens` tokens in scattered pages; the last rows[b] of each are the rows of the call (0: none)."""

    def __init__(self, lens, rows, H, G, D, V, page, dtype, seed=0, spread=1.0):
        from lit_llama import kv4

        g = self.g = np.random.default_rng(seed)
        self.lens, self.rows, self.H, self.dtype, self.page = lens, rows, H, dtype, page
        self.lay = lay = kv4.Layout(G, D, V, page)
        need = [-(-n // page) for n in lens]
        pages = sum(need) + 3
        order = list(g.permutation(pages))
        B = len(lens)
        table = np.full((B + 2, max(need + [1]) + 1), -1)
        slots = g.permutation(B + 2)[:B]
        self.pool = lay.pool(pages)
        # places nobody wrote hold NaN pairs
        page_bytes = page * (O.width(D) + O.width(V)) // 2
        self.pool[:, :, page_bytes:] = 0xFF
        self.k, self.v = [], []
        for b, n in enumerate(lens):
            ids = [order.pop() for _ in range(need[b])]
            table[slots[b], :need[b]] = ids
            k, kd = rounded(keys(g, n, G, D), torch.bfloat16)
            v, vd = rounded(g.standard_normal((n, G, V)), torch.bfloat16)
            if n:
                kv4.write(self.pool, lay, kd, vd, ints([ids[t // page] * page + t % page for t in range(n)]))
            self.k.append(O.stands_for(k))
            self.v.append(O.stands_for(v))
        self.table, self.slot = ints(table), ints(slots)
        self.M = sum(rows)
        self.pos = [n - r + i for n, r in zip(lens, rows) for i in range(r)]
        self.seq = [b for b, r in enumerate(rows) for _ in range(r)]
        self.q, self.qd = rounded(spread * g.standard_normal((self.M, H * D)), dtype)
        self.gate, self.gated = rounded(g.standard_normal((self.M, H)), dtype)

    def work(self, per):
        out, first = [], 0
        for b, r in enumerate(self.rows):
            out += [[first + j, min(per, r - j), b] for j in range(0, r, per)]
            first += r
        return ints(out)

    def want(self, scale=None, sink=False, gate=False):
        D, V, H = self.lay.dim, self.lay.vdim, self.H
        scale = D ** -0.5 if scale is None else scale
        y, tol = np.zeros((self.M, H, V)), np.zeros((self.M, H, 1))
        half = float(torch.finfo(self.dtype).eps) / 2
        terms = 2.0 ** -16 if self.dtype == torch.bfloat16 else 2.0 ** -24
        R = H // self.lay.kv_heads
        for m in range(self.M):
            b, p = self.seq[m], self.pos[m]
            q = self.q[m].reshape(1, H, D)
            y[m] = O.attend(q, self.k[b], self.v[b], [p], scale, sink, self.gate[m][None] if gate else None)[0]
            if p < 0:
                continue
            for h in range(H):
                k, v = self.k[b][:p + 1, h // R], self.v[b][:p + 1, h // R]
                ks, vs = np.abs(k).max() + 31 * (k.max() - k.min()) / 15, np.abs(v).max() + 31 * (v.max() - v.min()) / 15
                e = (D + 8) * 2.0 ** -24 * scale * ks * np.abs(q[0, h]).sum()
                s = k @ q[0, h] * scale
                spread = max(s.max(), 0.0) - min(s.min(), 0.0)
                tol[m, h] = np.abs(v).max() * (np.expm1(2 * e) + 2.0 ** -21 + 2.0 ** -22 * spread) + vs * (terms + (p + 1) * 2.0 ** -24)
        return y.reshape(self.M, -1), (tol + (half + 2.0 ** -21) * np.abs(y)).reshape(self.M, -1)

    def run(self, per=None, q=None, **kw):
        from lit_llama import kv4

        if kw.pop("gate", False):
            kw["gate"] = self.gated
        if per is not None:
            kw.update(work=self.work(per), rows=per)
        return kv4.attend(self.qd if q is None else q, self.pool, self.lay, self.table, self.slot, ints(self.pos), **kw)

    def check(self, y, **kw):
        want, tol = self.want(**kw)
        off = np.abs(y.double().cpu().numpy().reshape(want.shape) - want)
        assert (off <= tol).all(), f"{(off > tol).sum()} of {off.size} outside, the worst {np.max(off / np.maximum(tol, 1e-300)):.3g} of its bound"


SIZES = [(4, 2, 64, 64, 16), (8, 2, 128, 128, 64), (2, 2, 128, 128, 128), (6, 3, 78, 78, 32), (20, 1, 96, 64, 16), (5, 1, 40, 200, 64), (3, 3, 256, 256, 16),
         (34, 2, 130, 66, 256), (2, 1, 1, 1, 16), (4, 4, 33, 17, 128), (4, 2, 200, 90, 32), (2, 2, 64, 160, 16), (2, 1, 160, 48, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,G,D,V,page", SIZES)
def test_steps(hip, dtype, H, G, D, V, page):
    """One row per sequence: a first token, ends inside a tile and a page, exactly on them, one behind; an idle place."""
    c = Case([1, 2, 15, 16, 17, 63, 64, 65, 0, 128, 257, 300], [1] * 12, H, G, D, V, page, dtype, seed=D + V)
    c.check(c.run())
    c.check(c.run(scale=0.05, sink=True, gate=True), scale=0.05, sink=True, gate=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,G,D,V,page", SIZES)
@pytest.mark.parametrize("per", [1, 3, 40, 200])
def test_rows_of_several_tokens(hip, dtype, H, G, D, V, page, per):
    """Prompt rows and portions behind earlier tokens in items of every size; a sequence without rows between."""
    c = Case([5, 40, 1, 33, 150], [5, 7, 1, 0, 70], H, G, D, V, page, dtype, seed=H)
    c.check(c.run(per))
    c.check(c.run(per, sink=True, gate=True), sink=True, gate=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1023, 4096, 20001])
def test_long_sequences(hip, dtype, n):
    """Key ranges over several workgroups, and queries with a few keys that win."""
    c = Case([n, 700], [1, 1], 8, 2, 128, 128, 64, dtype, seed=n, spread=3.0)
    c.check(c.run())
    c = Case([n, 700], [3, 2], 4, 2, 64, 64, 16, dtype, seed=n)
    c.check(c.run(4, sink=True), sink=True)


@pytest.mark.parametrize("per", [None, 2, 40])
def test_fp32_weights_keep_their_bits(hip, per):
    """Heads of one value and a small scale, whose scores are nearly exact, over three keys each: what is left is the weights, 22 bits each. (Terms
    that did not add up to the weight left one row in a thousand off by 2^-11 of one.)"""
    c = Case([3] * 400, [1 if per is None else 3] * 400, 8, 1, 1, 64, 16, torch.float32, seed=12)
    c.check(c.run(per, scale=0.02), scale=0.02)


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_prompt(hip, dtype):
    c = Case([900, 130], [333, 130], 4, 2, 128, 128, 64, dtype, seed=8)
    c.check(c.run(64, gate=True), gate=True)
    c = Case([700], [700], 3, 1, 64, 64, 32, dtype, seed=9)
    c.check(c.run(42, sink=True), sink=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,V", [(64, 64), (128, 128), (120, 64), (40, 100)])
def test_many_prompts(hip, dtype, D, V):
    """More workgroups than half the CUs, which take 128 columns each where fewer take 64: portions of 17 and 18 rows of 80 sequences, and the same
    rows in calls of 10 sequences."""
    g = np.random.default_rng(D)
    rows = [17 + i % 2 for i in range(80)]
    c = Case([int(r + n) for r, n in zip(rows, g.integers(0, 190, 80))], rows, 8, 2, D, V, 32, dtype, seed=V)
    y = c.run(32, gate=True)
    c.check(y, gate=True)
    from lit_llama import kv4

    work, pos = c.work(32), ints(c.pos)
    z = torch.full_like(y, float("nan"))
    for i in range(0, 80, 10):
        kv4.attend(c.qd, c.pool, c.lay, c.table, c.slot, pos, work=work[i:i + 10].contiguous(), rows=32, gate=c.gated, out=z)
    c.check(z, gate=True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_see_nothing(hip, dtype):
    """pos < 0 (also below -1), slots outside the tables and pages outside the pool: zero rows, with and without ranges and a sink; a gap in
    the middle of a table hides its own tokens only."""
    c = Case([600, 600, 40], [1, 1, 1], 4, 2, 64, 64, 16, dtype)
    from lit_llama import kv4

    pos = ints([-1, 599, -7])
    for sink in (False, True):
        y = kv4.attend(c.qd, c.pool, c.lay, c.table, c.slot, pos, sink=sink)
        assert not y[0].any() and not y[2].any() and y[1].any()
    bad = ints([c.slot[0].item(), -1, 5])
    y = kv4.attend(c.qd, c.pool, c.lay, c.table, bad, ints(c.pos))
    assert y[0].any() and not y[1].any() and not y[2].any()
    t = c.table.clone()
    t[c.slot[0].item()] = 1 << 20
    t[c.slot[1].item(), 7] = -1
    y = kv4.attend(c.qd, c.pool, c.lay, t, c.slot, ints(c.pos))
    assert not y[0].any()
    keep = [j for j in range(600) if not 7 * 16 <= j < 8 * 16]
    c.k[1], c.v[1] = c.k[1][keep], c.v[1][keep]
    c.pos[1] = len(keep) - 1
    want, tol = c.want()
    assert (np.abs(y.double().cpu().numpy() - want) <= tol)[1:].all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("per", [None, 8])
def test_what_stands_behind_a_row_is_not_read(hip, dtype, per):
    """NaN keys and values at later positions of the same page do not reach a row, in rows of one call either; NaN at a visible one does."""
    from lit_llama import kv4

    c = Case([30], [1] if per is None else [6], 2, 1, 64, 64, 32, dtype)
    at = int(c.table[c.slot[0].item(), 0]) * 32
    nan = torch.full((1, 1, 64), float("nan"), dtype=dtype, device="cuda")
    if per is None:
        kv4.write(c.pool, c.lay, nan, nan, ints([at + 30]))
        c.check(c.run())
        kv4.write(c.pool, c.lay, nan, nan, ints([at + 11]))
        assert c.run().isnan().all()
    else:
        kv4.write(c.pool, c.lay, nan, nan, ints([at + 27]))  # the rows are positions 24 .. 29
        y = c.run(per)
        assert y[3:].isnan().all()
        want, tol = c.want()
        assert (np.abs(y.double().cpu().numpy() - want) <= tol)[:3].all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_behind_a_prompts_row(hip, dtype):
    """The same among prompt rows, which share their tiles: NaN at position 90 reaches rows 90 .. 129 and no others."""
    from lit_llama import kv4

    c = Case([130], [130], 2, 1, 64, 64, 32, dtype)
    at = int(c.table[c.slot[0].item(), 2]) * 32 + 90 - 64
    nan = torch.full((1, 1, 64), float("nan"), dtype=dtype, device="cuda")
    kv4.write(c.pool, c.lay, nan, nan, ints([at]))
    y = c.run(64)
    assert y[90:].isnan().all()
    want, tol = c.want()
    assert (np.abs(y.double().cpu().numpy() - want) <= tol)[:90].all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_tile_of_nan_behind_a_prompts_row(hip, dtype):
    """Positions 64 .. 127 all NaN, a tile of keys without one scale: rows 0 .. 63 of the same item do not see them."""
    from lit_llama import kv4

    c = Case([130], [130], 2, 1, 64, 64, 64, dtype)
    at = int(c.table[c.slot[0].item(), 1]) * 64
    nan = torch.full((64, 1, 64), float("nan"), dtype=dtype, device="cuda")
    kv4.write(c.pool, c.lay, nan, nan, ints(range(at, at + 64)))
    y = c.run(64)
    assert y[64:].isnan().all()
    want, tol = c.want()
    assert (np.abs(y.double().cpu().numpy() - want) <= tol)[:64].all()


def put(c, b, places, k=None, v=None):
    """Keys, values (t, G, n) of sequence b at these places replaced, in the cache and in what is expected."""
    from lit_llama import kv4

    row = c.table[c.slot[b].item()].tolist()
    k = rounded(c.k[b][places] if k is None else k, torch.float32)
    v = rounded(c.v[b][places] if v is None else v, torch.float32)
    kv4.write(c.pool, c.lay, k[1], v[1], ints([row[t // c.page] * c.page + t % c.page for t in places]))
    c.k[b][places], c.v[b][places] = O.stands_for(k[0]), O.stands_for(v[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [64, 128])
@pytest.mark.parametrize("rows,per", [(6, 8), (130, 64)])
def test_large_values_behind_a_row(hip, dtype, n, rows, per):
    """A value 2^30 times the others: rows before its position keep every digit of theirs, in one item with the rows that see it."""
    c = Case([150], [rows], 2, 1, n, n, 32, dtype, seed=n)
    put(c, 0, [146], v=c.g.standard_normal((1, 1, n)) * 2.0 ** 30)
    c.check(c.run(per))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("low", [[300], list(range(128)), list(range(3, 690, 7))])
@pytest.mark.parametrize("rows,per", [(1, None), (4, 8), (130, 64)])
def test_large_values_of_keys_that_do_not_count(hip, dtype, low, rows, per):
    """Seen keys whose scores are 60 and more below the others', e^-60 of their weights, with values 2^30 times the others': less than 2^-56 of a
    result, so it is expected as if they were not there (and the others' weights, relative to the largest value and score among them, as precise)."""
    c = Case([820], [rows], 2, 1, 64, 64, 64, dtype, seed=4)
    q = c.q.reshape(rows, 2, 64)
    q[:, :, 0] = 20
    c.q, c.qd = rounded(q.reshape(rows, -1), dtype)
    every = np.arange(820)
    put(c, 0, every, k=np.where(np.arange(64) == 0, np.clip(c.k[0], -2, 2), c.k[0]))
    put(c, 0, low, k=np.broadcast_to(np.where(np.arange(64) == 0, -40.0, 0.0), (len(low), 1, 64)),
        v=c.g.standard_normal((len(low), 1, 64)) * 2.0 ** 30)
    y = c.run(per)
    s = np.einsum("mhd,td->mht", c.q.reshape(rows, 2, 64), c.k[0][:, 0]) / 8
    keep = np.setdiff1d(every, low)
    first = 820 - rows
    assert (s[:, :, keep[keep <= first]].max(2) - s[:, :, low].max(2) > 60).all()
    c.k[0], c.v[0] = c.k[0][keep], c.v[0][keep]
    c.pos = [p - len(low) for p in c.pos]
    c.check(y)


@pytest.mark.parametrize("dtype", DTYPES)
def test_pages_far_into_a_large_pool(hip, dtype):
    """Places whose bytes lie past 2^32: rows written, read and attended to as at the pool's beginning."""
    from lit_llama import kv4

    lay = kv4.Layout(1, 128, 128, 64)
    n = (1 << 32) // lay.block_bytes() + 40
    pool = torch.empty(n, 1, lay.block_bytes(), dtype=torch.uint8, device="cuda")
    g = np.random.default_rng(1)
    L = 700
    k, v = (rounded(x, dtype)[1] for x in (keys(g, L, 1, 128), g.standard_normal((L, 1, 128))))
    q = rounded(g.standard_normal((40, 4 * 128)), dtype)[1]
    out = []
    for ids in (range(0, 11), range(n - 11, n)):
        place = ints([ids[t // 64] * 64 + t % 64 for t in range(L)])
        kv4.write(pool, lay, k, v, place)
        a = kv4.read(pool, lay, place, dtype)
        table = ints([list(ids)])
        y = kv4.attend(q[:1], pool, lay, table, ints([0]), ints([L - 1]))
        z = kv4.attend(q, pool, lay, table, ints([0]), ints(range(L - 40, L)), work=ints([[0, 40, 0]]), rows=40)
        out.append((*a, y, z))
    for a, b in zip(*out):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [128, 256])
def test_wide_heads_in_a_graph(hip, dtype, D):
    """Kernels of more than 64 KiB of shared memory, never launched before the capture of their call: a step and prompt rows."""
    c = Case([700, 300], [1, 1], 4, 2, D, D, 64, dtype, seed=D)
    p = Case([200], [150], 4, 2, D, D, 64, dtype, seed=D + 1)
    work, pos, ppos, graph = p.work(64), ints(c.pos), ints(p.pos), torch.cuda.CUDAGraph()
    from lit_llama import kv4

    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = kv4.attend(c.qd, c.pool, c.lay, c.table, c.slot, pos)
        z = kv4.attend(p.qd, p.pool, p.lay, p.table, p.slot, ppos, work=work, rows=64)
    for _ in range(3):
        y.fill_(7.0)
        z.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        c.check(y)
        p.check(z)


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompt_rows_in_a_graph(hip, dtype):
    """Rows behind a long cache, in key ranges that a second launch joins, captured and replayed over new queries and lengths."""
    from lit_llama import kv4

    c = Case([2600], [40], 8, 2, 64, 64, 64, dtype, seed=3)
    work, pos, q = c.work(40), ints(c.pos), c.qd.clone()
    assert kv4.splits(c.lay, 8, 1, 40, 2600, dtype)[0] > 1
    kv4.attend(q, c.pool, c.lay, c.table, c.slot, pos, work=work, rows=40)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = kv4.attend(q, c.pool, c.lay, c.table, c.slot, pos, work=work, rows=40)
    for turn in range(3):
        first = [2559, 100, -3][turn]
        c.pos = [first + i for i in range(40)]
        c.q, qd = rounded(np.random.default_rng(turn).standard_normal(c.q.shape), dtype)
        q.copy_(qd)
        pos.copy_(ints(c.pos))
        graph.replay()
        torch.cuda.synchronize()
        c.check(y)
        assert torch.equal(y, kv4.attend(qd, c.pool, c.lay, c.table, c.slot, ints(c.pos), work=work, rows=40))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_rows_and_outputs(hip, dtype):
    """Queries and gates out of packed projections at odd columns, into a wider output; rows of no item are left as they were."""
    c = Case([100, 41, 7], [1, 1, 1], 6, 2, 64, 64, 16, dtype, seed=2)
    wide = torch.zeros(3, 6 * 64 + 6 + 5, dtype=dtype, device="cuda")
    wide[:, 3:3 + 384] = c.qd
    wide[:, 387:393] = c.gated
    out = torch.full((3, 400), 7.0, dtype=dtype, device="cuda")
    from lit_llama import kv4

    kv4.attend(wide[:, 3:387], c.pool, c.lay, c.table, c.slot, ints(c.pos), gate=wide[:, 387:393], out=out[:, 5:389])
    c.check(out[:, 5:389], gate=True)
    assert (out[:, :5] == 7).all() and (out[:, 389:] == 7).all()
    out.fill_(7.0)
    kv4.attend(c.qd, c.pool, c.lay, c.table, c.slot, ints(c.pos), out=out[:, :384], work=ints([[2, 1, 2], [0, 0, 0], [0, 1, 0]]), rows=1)
    want, tol = c.want()
    assert (np.abs(out[:, :384].double().cpu().numpy() - want) <= tol)[[0, 2]].all() and (out[1] == 7).all()
    # items that name no rows of the call
    out.fill_(7.0)
    kv4.attend(c.qd, c.pool, c.lay, c.table, c.slot, ints(c.pos), out=out[:, :384], work=ints([[3, 1, 0], [-1, 1, 0], [0, 1, 3], [2, 2, 0], [0, -4, 0]]), rows=2)
    assert (out == 7).all()


def test_kept_counters_and_graphs(hip):
    """Counters that a program keeps, over calls of different sizes; a captured call replayed over new rows and lengths, with eager
    calls between."""
    from lit_llama import kv4

    c = Case([3000, 2500], [1, 1], 8, 2, 128, 128, 64, torch.bfloat16, seed=4)
    count = torch.zeros(64, dtype=torch.int32, device="cuda")
    q, pos = c.qd.clone(), ints(c.pos)
    kv4.attend(q, c.pool, c.lay, c.table, c.slot, pos, count=count)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = kv4.attend(q, c.pool, c.lay, c.table, c.slot, pos, count=count)
    g = np.random.default_rng(0)
    for turn in range(4):
        c.pos = [int(g.integers(0, 3000)), int(g.integers(-1, 2500))]
        c.q, qd = rounded(g.standard_normal(c.q.shape), torch.bfloat16)
        q.copy_(qd)
        pos.copy_(ints(c.pos))
        graph.replay()
        torch.cuda.synchronize()
        c.check(y)
        e = kv4.attend(qd, c.pool, c.lay, c.table, c.slot, ints(c.pos), count=count)
        assert torch.equal(e, y) and not count.any()
        small = Case([700], [1], 2, 2, 64, 64, 16, torch.float32, seed=turn)
        small.check(small.run(count=count))
        assert not count.any()


def test_two_streams(hip):
    """Calls on two streams at once, each with counters of its own."""
    a = Case([5000, 4000], [1, 1], 8, 2, 128, 128, 64, torch.bfloat16, seed=5)
    b = Case([2500], [1], 4, 4, 64, 64, 16, torch.float32, seed=6)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    ya, yb = [], []
    for _ in range(10):
        with torch.cuda.stream(s1):
            ya.append(a.run())
        with torch.cuda.stream(s2):
            yb.append(b.run())
    torch.cuda.synchronize()
    a.check(ya[0])
    b.check(yb[0])
    assert all(torch.equal(y, ya[0]) for y in ya) and all(torch.equal(y, yb[0]) for y in yb)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 64])
def test_a_serving_run(hip, dtype, page):
    """The operators together: unequal prompts, steps, a portion, one request ending and another taking its slot and pages."""
    from lit_llama import kv4, pages

    g = np.random.default_rng(page)
    H, G, D, V = 8, 2, 64, 64
    lay = kv4.Layout(G, D, V, page)
    n_pages = 400 // page + 6
    table, seen = ints(np.full((4, 300 // page + 1), -1)), ints([0] * 4)
    free, nfree, fault = ints(g.permutation(n_pages)), ints([n_pages]), ints([0])
    pool = lay.pool(n_pages)
    keep = {s: ([], []) for s in range(4)}

    def call(slots, adds):
        M = sum(adds)
        r = pages.extend(table, seen, free, nfree, ints(slots), ints(adds), M, page, chunk=8, fault=fault)
        q, qd = rounded(g.standard_normal((M, H * D)), dtype)
        k, kd = rounded(keys(g, M, G, D), dtype)
        v, vd = rounded(g.standard_normal((M, G, V)), dtype)
        kv4.write(pool, lay, kd, vd, r.place)
        step = max(adds) == 1
        y = kv4.attend(qd, pool, lay, table, ints(slots), r.pos, work=None if step else r.work, rows=1 if step else 8)
        c = Case.__new__(Case)
        c.lay, c.H, c.dtype, c.M, c.q, c.seq, c.pos, c.k, c.v = lay, H, dtype, M, q, [], [], [], []
        row = 0
        for b, (s, n) in enumerate(zip(slots, adds)):
            keep[s][0].extend(O.stands_for(k[row:row + n]))
            keep[s][1].extend(O.stands_for(v[row:row + n]))
            c.k.append(np.array(keep[s][0]))
            c.v.append(np.array(keep[s][1]))
            c.pos += range(len(keep[s][0]) - n, len(keep[s][0]))
            c.seq += [b] * n
            row += n
        assert r.pos.tolist() == c.pos
        c.check(y)

    call([2, 0, 3], [37, 1, 90])
    for _ in range(3):
        call([0, 3, 2], [1, 1, 1])
    call([3, 0], [20, 65])
    assert int(pages.release(table, seen, free, nfree, ints([3]), page, fault)) == 0
    keep[3] = ([], [])
    call([1, 3], [64, 33])
    for _ in range(2):
        call([3, 1, 0, 2], [1, 1, 1, 1])
    assert int(fault) == 0
