"""Block tables and slot maps (csrc/pages.hip) against oracle/kv4_np.py's tables, kept on the host request by request."""
import numpy as np
import pytest
import torch

from oracle import kv4_np as O

pytestmark = pytest.mark.gpu


def ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32).cuda()


class Both:
    """The tables on the device and the oracle's."""

    def __init__(self, slots, width, pages, page, seed=0):
        g = np.random.default_rng(seed)
        free = g.permutation(pages)
        self.page, self.pages = page, pages
        self.want = O.Tables(np.full((slots, width), -1), [0] * slots, free, page)
        self.table, self.seen = ints(np.full((slots, width), -1)), ints([0] * slots)
        self.free, self.nfree = ints(free), ints([pages])
        self.fault = ints([0])

    def args(self):
        return self.table, self.seen, self.free, self.nfree

    def extend(self, slots, adds, extra=0, chunk=0, **kw):
        from lit_llama import pages

        M = sum(adds) + extra
        r = pages.extend(*self.args(), ints(slots), None if kw.pop("ones", False) else ints(adds), M, self.page, chunk=chunk, fault=self.fault, **kw)
        return r, M

    def check(self, slots, adds, extra=0, chunk=0, **kw):
        r, M = self.extend(slots, adds, extra, chunk, **kw)
        row0, seq, pos, place, work = self.want.extend(slots, adds, chunk)
        assert int(r.status) == 0 and int(self.fault) == 0
        assert r.row0.tolist() == row0
        for got, want in ((r.row_seq, seq), (r.pos, pos), (r.place, place)):
            assert got.tolist() == want + [-1] * (M - len(want))
        if chunk:
            assert r.work.tolist() == work + [[0, 0, 0]] * (M // chunk + len(slots) - len(work))
            assert r.item0.tolist() == [sum(-(-a // chunk) for a in adds[:b]) for b in range(len(adds) + 1)]
        assert r.seen.tolist() == [self.want.seen[s] for s in slots] and int(r.left) == len(self.want.free)
        self.same()
        return r

    def same(self):
        assert self.table.tolist() == self.want.table and self.seen.tolist() == self.want.seen
        n = int(self.nfree)
        assert n == len(self.want.free) and self.free.tolist()[:n] == self.want.free


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_calls_of_a_serving_loop(hip, page):
    """Prompts, steps, ends and new requests in turn: odd lengths, requests that add nothing, pages that fill exactly."""
    from lit_llama import pages

    g = np.random.default_rng(page)
    t = Both(9, 40, 300, page, seed=page)
    t.check([3], [1])
    t.check([4, 0, 7], [page, 2 * page + 1, 3], chunk=64)
    for turn in range(12):
        live = list(g.permutation(9)[:g.integers(1, 10)])
        if turn % 3 == 2:
            ends = live[:2]
            assert int(pages.release(*t.args(), ints(ends), page, t.fault)) == 0
            t.want.release(ends)
            t.same()
        adds = [int(a) for a in g.choice([0, 1, 1, 2, page - 1, page, page + 1, 2 * page], len(live))]
        t.check(live, adds, extra=int(g.integers(0, 5)) + (sum(adds) == 0), chunk=[0, 1, 7, 64][turn % 4])
        t.check(live, [1] * len(live), ones=True)


@pytest.mark.parametrize("B", [1, 63, 64, 65, 256, 1024, 1025, 4096])
def test_many_sequences(hip, B):
    g = np.random.default_rng(B)
    t = Both(B + 3, 9, 9 * (B + 3), 16, seed=B)
    slots = [int(s) for s in g.permutation(B + 3)[:B]]
    t.check(slots, [int(a) for a in g.integers(0, 30, B)], extra=3, chunk=8)
    t.check(slots, [1] * B, ones=True, extra=1)


@pytest.mark.parametrize("M", [4095, 4096, 4097, 8191, 8192, 8193, 30000])
def test_long_prompts(hip, M):
    """On both sides of the size from which the rows have a launch of their own."""
    t = Both(4, 4000, 8000, 16)
    t.check([2, 0], [M // 3, M - M // 3], chunk=64)
    t.check([0, 2, 3], [M, 0, 1], chunk=13)


def test_the_largest_tables(hip):
    """All 65,536 slots, the last of them in use."""
    t = Both(65536, 1, 70000, 16)
    slots = [65535, 0, 31, 32, 40000]
    t.check(slots, [16, 1, 2, 3, 4], chunk=2)
    t.check(slots[1:], [1] * 4)


def test_a_sequence_of_2_to_the_30_tokens(hip):
    """The longest there is: it stays in a call that adds nothing, takes no token more, and gives its pages back."""
    from lit_llama import pages

    width = 1 << 26
    table = torch.arange(width, dtype=torch.int32, device="cuda").view(1, width)
    seen, free, nfree, fault = ints([1 << 30]), torch.full((width,), -5, dtype=torch.int32, device="cuda"), ints([0]), ints([0])
    args = table, seen, free, nfree
    r = pages.extend(*args, ints([0]), ints([0]), 3, 16, fault=fault)
    assert int(r.status) == 0 and r.seen.tolist() == [1 << 30] and r.pos.tolist() == [-1] * 3
    r = pages.extend(*args, ints([0]), ints([1]), 3, 16)
    assert int(r.status) == pages.BAD_CALL and r.pos.tolist() == [-1] * 3 and seen.tolist() == [1 << 30]
    assert int(pages.release(*args, ints([0]), 16, fault=fault)) == 0 and fault.tolist() == [0]
    assert nfree.tolist() == [width] and seen.tolist() == [0]
    assert torch.equal(free, torch.arange(width, dtype=torch.int32, device="cuda")) and bool((table == -1).all())


def test_without_commit_the_same_call_again(hip):
    t = Both(4, 10, 30, 16)
    t.check([1, 2], [20, 5])
    a, _ = t.extend([2, 3, 1], [30, 1, 40], chunk=16, commit=False)
    assert int(t.nfree) == len(t.want.free) and t.seen.tolist() == t.want.seen
    b = t.check([2, 3, 1], [30, 1, 40], chunk=16)
    for n in ("row0", "item0", "row_seq", "pos", "place", "work", "seen", "left", "status"):
        assert torch.equal(getattr(a, n), getattr(b, n)), n


@pytest.mark.parametrize("what", ["pages", "twice", "slot", "low slot", "negative", "width", "rows"])
def test_calls_left_undone(hip, what):
    """Nothing changes, there are no rows, the status says why; a good call afterwards works and leaves the fault standing."""
    from lit_llama import pages

    t = Both(5, 4, 9, 16)
    t.check([0, 1], [40, 17])
    slots, adds, extra, status = [2, 0, 1], [30, 1, 2], 0, 2
    if what == "pages":
        adds, status = [64, 20, 40], 1
    elif what == "twice":
        slots = [2, 0, 2]
    elif what == "slot":
        slots = [2, 5, 1]
    elif what == "low slot":
        slots = [2, -1, 1]
    elif what == "negative":
        adds = [30, -1, 2]
    elif what == "width":
        adds = [65, 1, 2]
    elif what == "rows":
        extra = -1
    before = [x.clone() for x in t.args()]
    r, M = t.extend(slots, adds, extra, chunk=16)
    assert int(r.status) == status and int(t.fault) == status
    assert all(torch.equal(a, b) for a, b in zip(before, t.args()))
    for x in (r.row_seq, r.pos, r.place):
        assert x.tolist() == [-1] * M
    assert not r.work.any() and not r.row0.any() and not r.item0.any() and int(r.left) == len(t.want.free)
    if what != "pages" and what != "rows" and what != "width" and what != "negative":
        assert int(pages.release(*t.args(), ints(slots), 16, None)) == 2
        assert all(torch.equal(a, b) for a, b in zip(before, t.args()))
    t.fault.zero_()
    t.check([2, 0, 1], [16, 1, 2])


def test_a_stack_that_cannot_be(hip):
    from lit_llama import pages

    t = Both(2, 4, 9, 16)
    for n in (-1, 10):
        t.nfree.fill_(n)
        r, _ = t.extend([0], [3])
        assert int(r.status) == 2 and r.place.tolist() == [-1] * 3 and int(t.nfree) == n
        assert int(pages.release(*t.args(), ints([1]), 16)) == 2


def test_steps_in_a_captured_graph(hip):
    """A captured step extends its sequences at every replay, eager calls between them, until the stack is empty."""
    from lit_llama import pages

    t = Both(3, 8, 10, 16)
    t.check([0, 1, 2], [15, 31, 1])
    slot = ints([2, 0, 1])
    t.extend([0], [0], extra=1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = pages.extend(*t.args(), slot, None, 3, 16, chunk=1, fault=t.fault)
    for _ in range(20):
        graph.replay()
        row0, seq, pos, place, work = t.want.extend([2, 0, 1], [1, 1, 1], 1)
        assert r.pos.tolist() == pos and r.place.tolist() == place and r.work.tolist() == work + [[0, 0, 0]] * 3
        t.same()
    t.check([1], [5])
    while len(t.want.free):
        graph.replay()
        t.want.extend([2, 0, 1], [1, 1, 1])
        t.same()
    for _ in range(40):
        graph.replay()
    assert int(t.fault) == 1 and int(r.status) == 1 and r.place.tolist() == [-1] * 3 and int(t.nfree) == 0


def test_calls_without_rows(hip):
    """Sequences that add nothing and no room for rows: lengths and first rows come back all the same."""
    t = Both(3, 4, 9, 16)
    t.check([2, 0], [5, 16])
    r = t.check([0, 2, 1], [0, 0, 0], chunk=4)
    assert r.seen.tolist() == [16, 5, 0] and r.pos.numel() == 0


def test_on_another_stream(hip):
    t = Both(3, 8, 20, 16)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        t.check([1, 0], [40, 3], chunk=16)
