"""The paged 4-bit cache without a GPU: the oracle against plain loops, sizes, and calls that are refused before anything is launched."""
import numpy as np
import pytest
import torch

from oracle import kv4_np as O

EINVAL = 1000


def lib():
    from lit_llama import _build, _hip

    if not _hip.LIB_PATH.exists():
        _build.build()
    return _hip.lib()


def test_codes_of_one_vector_at_a_time():
    g = np.random.default_rng(0)
    for scale in (1.0, 1e-20, 1e20):
        x = (g.standard_normal((50, 24)) * scale + g.standard_normal((50, 1)) * 3 * scale).astype(np.float32)
        c, s, o = O.quantize(x)
        for i in range(50):
            lo = float(torch.tensor(float(x[i].min())).bfloat16())
            if lo > x[i].min():
                lo = float(torch.nextafter(torch.tensor(lo).bfloat16(), torch.tensor(-float("inf")).bfloat16()))
            st = float(torch.tensor((float(x[i].max()) - lo) / 15).bfloat16())
            assert o[i] == lo and s[i] == st
            want = [min(15, max(0, round((float(v) - lo) / st))) for v in x[i]]
            assert c[i].tolist() == want
            # half a step, and 15 steps' rounding at the top
            assert np.abs(c[i] * st + lo - x[i]).max() <= st * (0.5 + 15 * 2.0 ** -8)


def test_vectors_without_a_code():
    x = np.zeros((4, 8), np.float32)
    x[0, 1], x[1, 2], x[2, 3] = np.nan, np.inf, -3.4e38
    c, s, o = O.quantize(x)
    assert np.isnan(s[:3]).all() and np.isnan(o[:3]).all() and s[3] == o[3] == 0 and not c.any()


def test_bf16_bits():
    x = np.random.default_rng(1).standard_normal(1000).astype(np.float32) * 10
    assert np.array_equal(O.from_bits(O.bf16_bits(x)), torch.tensor(x).bfloat16().double().numpy())
    f = O.from_bits(O.floor_bits(x))
    assert (f <= x).all() and (x - f < np.abs(x) * 2.0 ** -7).all()


def test_block_bytes():
    L = lib()
    for page in (16, 32, 64, 128, 256):
        for d, v in ((1, 1), (64, 64), (65, 64), (78, 128), (128, 129), (256, 200)):
            assert L.llj_kv4_block_bytes(page, d, v) == len(O.pack(np.zeros((1, d)), np.zeros((1, v)), page)) == page * ((O.width(d) + O.width(v)) // 2 + 8)
    for bad in ((0, 64, 64), (24, 64, 64), (8, 64, 64), (512, 64, 64), (64, 0, 64), (64, 257, 64), (64, 64, 0), (64, 64, 257)):
        assert L.llj_kv4_block_bytes(*bad) == 0
    from lit_llama import kv4

    with pytest.raises(ValueError):
        kv4.Layout(2, 64, 300, 64).block_bytes()
    with pytest.raises(ValueError):
        kv4.Layout(0, 64, 64, 64).block_bytes()
    assert L.llj_kv4_part_width(64) == 68 and L.llj_kv4_part_width(78) == 132 and L.llj_kv4_part_width(256) == 260


def test_tiles_and_ranges():
    from lit_llama import kv4

    L = lib()
    def tiles(heads, kv_heads, rows, dim=64, vdim=64, dt=0):
        return L.llj_kv4_tiles(heads, kv_heads, dim, vdim, rows, dt)

    assert tiles(8, 2, 1) == 2 and tiles(8, 2, 5) == 4 and tiles(34, 2, 1) == 4
    assert tiles(8, 2, 32) == 2 and tiles(8, 2, 33) == 4 and tiles(8, 2, 32, dt=1) == 4 and tiles(8, 2, 32, vdim=200) == 4
    assert tiles(8, 3, 1) == 0 and tiles(0, 1, 1) == 0 and tiles(8, 2, 0) == 0 and tiles(65535, 1, 65535) == 0 and tiles(8, 2, 1, dim=300) == 0
    lay = kv4.Layout(8, 128, 128, 64)
    for items, keys in ((1, 10), (1, 300), (1, 1 << 20), (8, 4096), (64, 8192), (4096, 1 << 20)):
        n, need = kv4.splits(lay, 32, items, 1, keys)
        assert 1 <= n <= 64 and (n == 1 or n * kv4.RANGE < keys + kv4.RANGE) and need == items * 8
    for items, rows, keys in ((1, 32, 64), (1, 32, 1000), (1, 17, 1 << 20), (16, 32, 512), (16, 32, 60000), (64, 32, 4096), (5000, 200, 1 << 20)):
        n, need = kv4.splits(lay, 32, items, rows, keys)
        assert 1 <= n <= min(64, -(-keys // 64)) and need == 0 and (n == 1 or n * items * 8 <= kv4.WGS)
    assert kv4.splits(lay, 32, 1, 32, 1 << 20)[0] == 64 and kv4.splits(lay, 32, 16, 32, 512)[0] == 1


P = 4096  # an address that nothing is read from: the calls below end at their checks


def test_pages_refuse():
    good = dict(slot=P, add=P, B=2, seen=P, slots=4, table=P, ldt=8, free=P, nfree=P, cap=9, page=16, commit=1, row0=P, item0=P, row_seq=P, pos=P, place=P,
                M=5, work=P, nwork=3, chunk=4, after=P, left=P, status=P, fault=None, stream=None)
    bad = [dict(slot=None), dict(B=0), dict(B=4097), dict(seen=None), dict(slots=0), dict(slots=65537), dict(table=None), dict(ldt=0), dict(ldt=1 << 27),
           dict(free=None), dict(nfree=None), dict(cap=0), dict(cap=1 << 27), dict(page=0), dict(page=8), dict(page=48), dict(page=512), dict(row0=None),
           dict(item0=None), dict(row_seq=None), dict(pos=None), dict(place=None), dict(M=-1), dict(M=(1 << 28) + 1), dict(work=None), dict(nwork=-1),
           dict(chunk=-1), dict(after=None), dict(left=None), dict(status=None)]
    for b in bad:
        assert lib().llj_pages_extend(*{**good, **b}.values()) == EINVAL, b
    good = dict(slot=P, B=2, seen=P, slots=4, table=P, ldt=8, free=P, nfree=P, cap=9, page=16, status=P, fault=None, stream=None)
    for b in [dict(slot=None), dict(B=0), dict(B=5000), dict(seen=None), dict(slots=0), dict(table=None), dict(ldt=0), dict(free=None), dict(nfree=None),
              dict(cap=0), dict(page=17), dict(status=None)]:
        assert lib().llj_pages_release(*{**good, **b}.values()) == EINVAL, b


def test_rows_refuse():
    good = dict(k=P, ldk=64, hk=32, v=P, ldv=64, hv=32, place=P, M=3, G=2, D=32, V=32, dt=0, pool=P, pages=4, page=16, stream=None)
    bad = [dict(k=None), dict(v=None), dict(place=None), dict(M=-1), dict(G=0), dict(G=5000), dict(D=0), dict(D=257), dict(V=0), dict(V=300), dict(dt=2),
           dict(pool=None), dict(pool=P + 8), dict(pages=0), dict(pages=1 << 27), dict(page=20), dict(ldk=1 << 41), dict(hv=1 << 62), dict(M=(1 << 25) + 1)]
    for b in bad:
        a = {**good, **b}
        assert lib().llj_kv4_write(*a.values()) == EINVAL, b
        assert lib().llj_kv4_read(*[a[n] for n in ("pool", "pages", "page", "place", "M", "G", "D", "V", "dt", "k", "ldk", "hk", "v", "ldv", "hv", "stream")]) == EINVAL, b
    assert lib().llj_kv4_write(*{**good, "M": 0}.values()) == 0


def test_preparation_refuses():
    good = dict(inp=P, ld=256, oq=0, ok=128, ov=192, turns=P, rot=32, norm=1, eps=1e-5, pos=P, place=P, pool=P, pages=4, page=16, first=None, lam=None,
                ldf=0, M=3, heads=4, kv_heads=2, dim=32, vdim=32, dt=0, stream=None)
    bad = [dict(inp=None), dict(ld=255), dict(oq=-1), dict(ok=200), dict(ov=193), dict(turns=None), dict(rot=33), dict(rot=34), dict(pos=None),
           dict(place=None), dict(pool=None), dict(pool=P + 8), dict(pages=0), dict(page=24), dict(lam=P), dict(first=P, ldf=63), dict(M=0),
           dict(M=(1 << 23) + 1), dict(heads=3), dict(heads=0), dict(kv_heads=0), dict(dim=0), dict(dim=257), dict(vdim=0), dict(vdim=300), dict(dt=2),
           dict(heads=200, kv_heads=200, dim=256, vdim=256, ld=1 << 20, ok=1 << 18, ov=1 << 19)]
    for b in bad:
        assert lib().llj_gqa_prep_kv4(*{**good, **b}.values()) == EINVAL, b


def test_attention_refuses():
    good = dict(q=P, ldq=256, gate=None, ldg=0, work=P, items=2, rows=2, pos=P, slot=P, B=2, table=P, slots=4, ldt=8, pool=P, pages=4, page=16, part=P,
                count=P, nsplit=2, y=P, ldy=256, M=4, heads=4, kv_heads=2, dim=64, vdim=64, scale=1.0, sink=0, dt=0, stream=None)
    bad = [dict(q=None), dict(ldq=255), dict(gate=P, ldg=3), dict(items=-1), dict(rows=0), dict(rows=70000), dict(pos=None), dict(slot=None), dict(B=0),
           dict(table=None), dict(slots=0), dict(ldt=0), dict(ldt=1 << 27), dict(pool=None), dict(pool=P + 4), dict(pages=0), dict(page=30), dict(part=None),
           dict(count=None), dict(part=P + 4), dict(nsplit=0), dict(nsplit=65), dict(y=None), dict(ldy=255), dict(M=-1), dict(heads=0), dict(heads=3),
           dict(kv_heads=0), dict(dim=0), dict(dim=257), dict(vdim=0), dict(vdim=260), dict(dt=2), dict(work=None), dict(work=None, rows=1, items=5, M=5),
           dict(work=None, rows=1, items=3, M=2, B=4), dict(heads=70000, kv_heads=35000, ldq=1 << 30),
           dict(items=1 << 23)]
    for b in bad:
        assert lib().llj_kv4_attend(*{**good, **b}.values()) == EINVAL, b
    assert lib().llj_kv4_attend(*{**good, "items": 0}.values()) == 0


def test_host_tensors_are_refused():
    from lit_llama import _hip, kv4, pages

    lib()
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(_hip.HipError):
        pages.extend(i(2, 3), i(2), i(5), i(1), i(1), None, 1, 16)
    with pytest.raises(ValueError):
        pages.extend(i(2, 3).long(), i(2), i(5), i(1), i(1), None, 1, 16)
    with pytest.raises(_hip.HipError):
        pages.release(i(2, 3), i(2), i(5), i(1), i(1), 16)
    lay = kv4.Layout(2, 64, 64, 16)
    pool = lay.pool(3, device="cpu")
    x = torch.zeros(2, 128)
    for f in (lambda: kv4.write(pool, lay, x, x, i(2)), lambda: kv4.read(pool, lay, i(2)),
              lambda: kv4.attend(x, pool, lay, i(2, 3), i(2), i(2))):
        with pytest.raises(_hip.HipError):
            f()
    with pytest.raises(ValueError):
        kv4.read(pool[:, :1], lay, i(2))
    with pytest.raises(ValueError):
        kv4.read(pool.int(), lay, i(2))
    with pytest.raises(ValueError):
        kv4.read(lay.pool(3, device="cpu").transpose(0, 1), lay, i(2))


def test_states_without_such_a_cache():
    from types import SimpleNamespace

    from lit_llama.state import SequenceState

    model = SimpleNamespace(mixers=[SimpleNamespace(ring_window=lambda: 8), SimpleNamespace(ring_window=lambda: None)])
    with pytest.raises(ValueError, match="4 bits"):
        SequenceState(model, 1, None, "int4")
    with pytest.raises(ValueError, match="int4"):
        SequenceState(model, 1, None, "int8")


def test_rows_of_an_item():
    from lit_llama import kv4

    lay = kv4.Layout(8, 128, 128, 64)
    assert [kv4.item_rows(lay, 32, n) for n in (1, 16, 17, 5000)] == [4, 4, 32, 32]
    assert kv4.item_rows(kv4.Layout(1, 200, 64, 16), 20, 500) == 6 and kv4.item_rows(kv4.Layout(1, 64, 64, 16), 300, 1) == 1
    for heads in range(1, 301):  # prompt rows' items are prompt rows
        per = kv4.item_rows(kv4.Layout(1, 64, 64, 16), heads, 1000)
        assert per * heads > kv4.FEW_COLUMNS and (per * heads <= 128 or per == 1)
