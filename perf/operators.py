"""The operators of a paged K / V cache in 4 bits, as a serving program calls them, over the sizes it calls them at.

  * "tables" -- block tables and slot maps of a call, made on the GPU from the requests' lengths (lit_llama.pages.extend);
  * "write"  -- rows of keys and values into the cache and what they stand for there (lit_llama.kv4.write and read);
  * "attend" -- grouped-query attention over the cache: one row per sequence, a few, or prompt rows (lit_llama.kv4.attend).

A vector x (a head's key or value) is held as codes c in 0 .. 15 with a bf16 scale s and offset o and stands for c s + o:
o the largest bf16 up to min x, s = (max x - o) / 15 rounded to float32 and then to bf16, c = (x - o) / s rounded to the nearest
(halves to even) and kept in 0 .. 15, all zero where s is. Sizes are those of this repository's models (heads of 64 and 128, 78 in
the 125M; 16 on 4 and 32 on 8 heads in the hybrid sizes; LLaMA's heads each with keys of their own).
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path.cwd() / "lit-llama-ja_amd"))  # the package of the tree this is run from

own = False
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
TABLE_ROWS = 64  # rows of a work item in the tables' cases


def listed() -> list:
    return [
        # a decode step of eight requests: launch latency is all there is
        _tables("tables-step", 8, 0, 1, 1000, 64),
        # a step in which some of 48 requests bring prompts of up to 1,500 tokens
        _tables("tables-prompts", 48, 9, 1500, 2001, 16),
        # a large serving batch: 2,048 requests with 64 tokens each on the average
        _tables("tables-large", 2048, 1024, 255, 4000, 128),
        # the rows of a decode step
        _write("write-step", 8, 8, 128, 128, 64, "bf16"),
        # prompts of the 1B model in single precision, an odd number of rows
        _write("write-prompts", 1003, 4, 128, 128, 64, "f32"),
        # a large prefill
        _write("write-large", 32768, 8, 128, 128, 64, "bf16"),
        # one user early in a chat with the 1B model
        _attend("step-chat", 1, 300, 1, 16, 4, 128, 64, "bf16"),
        # a batch of the 7B hybrid model, requests of 2,000 to 4,000 tokens, some places of the batch idle
        _attend("step-batch", 8, 4000, 1, 32, 8, 128, 64, "bf16", ragged=True, gate=True, sink=True, idle=True),
        # a large serving batch
        _attend("step-large", 64, 8192, 1, 32, 8, 128, 64, "bf16", ragged=True),
        # one long document, LLaMA's heads with keys of their own
        _attend("step-long", 1, 131071, 1, 32, 32, 128, 128, "bf16"),
        # prompts of several users on the 49M in single precision
        _attend("prompts-ragged", 6, 501, 501, 10, 10, 64, 16, "f32", ragged=True),
        # one long prompt of the 7B hybrid model
        _attend("prompt-long", 1, 4096, 4096, 32, 8, 128, 64, "bf16", gate=True, sink=True),
    ]


def _tables(name, batch, prompts, most, length, page) -> dict:
    """`batch` requests of up to `length` tokens so far; `prompts` of them bring up to `most` tokens, the others one."""
    return {"name": name, "kind": "tables", "batch": batch, "prompts": prompts, "most": most, "length": length, "page": page}


def _write(name, rows, kv_heads, dim, vdim, page, dtype) -> dict:
    return {"name": name, "kind": "write", "rows": rows, "kv_heads": kv_heads, "dim": dim, "vdim": vdim, "page": page, "dtype": dtype}


def _attend(name, batch, length, rows, heads, kv_heads, dim, page, dtype, ragged=False, gate=False, sink=False, idle=False) -> dict:
    """`batch` sequences of `length` tokens (ragged: half of that to all of it), the last `rows` of each the rows of this call
    (ragged prompts: all); idle: every fifth place of the batch has no tokens."""
    return {"name": name, "kind": "attend", "batch": batch, "length": length, "rows": rows, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "dtype": dtype, "ragged": ragged, "gate": gate, "sink": sink, "idle": idle}


def draw(rng) -> dict:
    """One more case of the listed ranges."""

    def spread(lo, hi):  # over the logarithm
        return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))

    page = rng.choice([16, 32, 64, 64, 128, 256])
    kind = rng.choice(["tables", "write", "step", "step", "step", "few", "prompt", "prompt"])
    if kind == "tables":
        batch = spread(1, 2048)
        prompts = rng.randint(0, batch // 2)
        most = spread(1, max(1, min(4096, 200000 // max(1, prompts))))
        case = _tables("", batch, prompts, most, spread(1, 8192), page)
    elif kind == "write":
        dim = rng.choice([64, 128, 128, 78, 96])
        case = _write("", spread(1, 16384), rng.choice([1, 2, 4, 8, 10]), dim, rng.choice([dim, dim, 64, 128]), page, rng.choice(["bf16", "bf16", "f32"]))
    else:
        heads, kv_heads = rng.choice([(16, 4), (32, 8), (32, 8), (32, 32), (10, 10), (12, 2), (8, 1), (20, 1)])
        dim = rng.choice([64, 128, 128, 128, 78, 96])
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        flags = {k: rng.random() < 0.4 for k in ("ragged", "gate", "sink")}
        if kind == "prompt":
            batch = spread(1, 8)
            length = spread(2, 4096 // batch)
            whole = rng.random() < 0.5
            rows = length if whole else spread(1, length)
            case = _attend("", batch, length, rows, heads, kv_heads, dim, page, dtype, **flags)
        else:
            batch = spread(1, 64)
            length = spread(4, min(131071, 2000000 // (batch * kv_heads)))
            rows = 1 if kind == "step" else min(length // 2, rng.randint(2, 8))
            case = _attend("", batch, length, rows, heads, kv_heads, dim, page, dtype, idle=rows == 1 and batch > 4 and rng.random() < 0.3, **flags)
    case.pop("name")
    return case


def _lengths(case) -> tuple:
    """(tokens, rows of this call) of every sequence of an attend case."""
    L, n = case["length"], case["rows"]
    tokens = [L - (b * 7919) % (L // 2 + 1) if case["ragged"] else L for b in range(case["batch"])]
    if case["idle"]:
        tokens = [0 if b % 5 == 3 else t for b, t in enumerate(tokens)]
    return tokens, [min(n, t) if n > 1 else 1 for t in tokens]


def _adds(case) -> list:
    """New tokens of every request of a tables case: prompts spread evenly over the batch."""
    B, P, most = case["batch"], case["prompts"], case["most"]
    adds = [1] * B
    for i in range(P):
        adds[i * B // P] = 1 + (i * 7919 + 13) % most
    return adds


def _width(n: int) -> int:
    """Values a vector takes in the cache: up to 64, 128 or 256."""
    return 64 if n <= 64 else 128 if n <= 128 else 256


def _views(pool, page, dim, vdim):
    """A pool (pages, heads, bytes) as key codes, value codes (.., page, width / 2) and key and value (scale, offset) pairs."""
    P, G = pool.shape[:2]
    kb, vb = page * _width(dim) // 2, page * _width(vdim) // 2
    parts = pool.split([kb, vb, 4 * page, 4 * page], -1)
    return (parts[0].view(P, G, page, -1), parts[1].view(P, G, page, -1), parts[2].view(torch.bfloat16).view(P, G, page, 2),
            parts[3].view(torch.bfloat16).view(P, G, page, 2))


# ------------------------------------------------------------------------------------------- inputs
def prepare(case, seed) -> dict:
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    kind = case["kind"]
    if kind == "tables":
        return _prepare_tables(case, g)
    page, G, D = case["page"], case["kv_heads"], case["dim"]
    dt = DTYPES[case["dtype"]]
    if kind == "write":
        V, M = case["vdim"], case["rows"]
        pages = -(-M // page) + 3
        place = torch.randperm(pages * page, generator=g, device=DEV)[:M].int() if M < 512 else torch.arange(M, device=DEV, dtype=torch.int32)
        pool = torch.zeros(pages, G, page * ((_width(D) + _width(V)) // 2 + 8), dtype=torch.uint8, device=DEV)
        k, v = _keys(M, G, D, g).to(dt), torch.randn(M, G, V, generator=g, device=DEV).to(dt)
        return {"kind": kind, "page": page, "pool": pool, "k": k, "v": v, "place": place}
    tokens, rows = _lengths(case)
    B, H = case["batch"], case["heads"]
    width = max(1, max(-(-t // page) for t in tokens))
    need = sum(-(-t // page) for t in tokens)
    pages = need + 2
    pool = _filled(pages, page, G, D, g)
    order = torch.randperm(pages, generator=g, device=DEV)[:need].int()
    table = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
    n = torch.tensor([-(-t // page) for t in tokens], device=DEV)
    table[torch.arange(width, device=DEV)[None] < n[:, None]] = order
    M = sum(rows)
    row_seq = torch.tensor([b for b, r in enumerate(rows) for _ in range(r)], dtype=torch.int32, device=DEV)
    pos = torch.tensor([t - r + i for t, r in zip(tokens, rows) for i in range(r)], dtype=torch.int32, device=DEV)
    R = H // G
    per, first, work = max(1, (16 if max(rows) * R <= 64 else 128) // R), 0, []
    for b, r in enumerate(rows):
        work += [[first + j, min(per, r - j), b] for j in range(0, r, per)]
        first += r
    qs = 1.5 * torch.randn(M, H * D, generator=g, device=DEV)
    gate = torch.randn(M, H, generator=g, device=DEV).to(dt) if case["gate"] else None
    return {"kind": kind, "page": page, "pool": pool, "table": table, "slot": torch.arange(B, dtype=torch.int32, device=DEV), "pos": pos,
            "row_seq": row_seq, "work": torch.tensor(work, dtype=torch.int32, device=DEV), "per": per, "q": qs.to(dt), "gate": gate,
            "sink": case["sink"], "H": H, "G": G, "D": D, "count": torch.zeros(64 * M * H, dtype=torch.int32, device=DEV),
            "keys": max(tokens), "rows": max(rows), "step": max(rows) == 1, "tokens": tokens, "new": rows}


def _keys(M, G, D, g):
    """Keys as trained models have them: channels of different spread around means of their own, a few of them large."""
    spread = 0.5 + torch.rand(G, D, generator=g, device=DEV)
    mean = torch.randn(G, D, generator=g, device=DEV) * (1.0 + 4.0 * (torch.rand(G, D, generator=g, device=DEV) < 0.03))
    return torch.randn(M, G, D, generator=g, device=DEV) * spread + mean


def _filled(pages, page, G, D, g):
    """A pool whose every place holds a key and a value."""
    pool = torch.zeros(pages, G, page * (_width(D) + 8), dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 26) // (page * G * D))
    for p in range(0, pages, step):
        n = min(step, pages - p) * page
        place = torch.arange(p * page, p * page + n, device=DEV)
        _store(pool, page, _keys(n, G, D, g).bfloat16(), torch.randn(n, G, D, generator=g, device=DEV).bfloat16(), place)
    return pool


def _prepare_tables(case, g) -> dict:
    B, page, length = case["batch"], case["page"], case["length"]
    adds = _adds(case)
    slots = B + 5
    slot = torch.randperm(slots, generator=g, device=DEV)[:B].int()
    seen = torch.randint(0, length + 1, (slots,), generator=g, device=DEV).int()
    add = torch.tensor(adds, dtype=torch.int32, device=DEV)
    width = -(-(length + max(adds)) // page)
    pages = slots * -(-length // page) + sum(-(-a // page) + 1 for a in adds) + 7
    ids = torch.randperm(pages, generator=g, device=DEV).int()
    have = (seen + page - 1) // page
    taken = torch.arange(width, device=DEV)[None] < have[:, None]
    table = torch.full((slots, width), -1, dtype=torch.int32, device=DEV)
    table[taken] = ids[:int(taken.sum())]
    left = ids[int(taken.sum()):]
    free = torch.zeros(pages, dtype=torch.int32, device=DEV)
    free[:left.numel()] = left
    nfree = torch.tensor([left.numel()], dtype=torch.int32, device=DEV)
    M = sum(adds)
    return {"kind": "tables", "page": page, "table": table, "seen": seen, "free": free, "nfree": nfree, "slot": slot, "add": add, "M": M,
            "nwork": M // TABLE_ROWS + B}


# ------------------------------------------------------------------------------------------- one pass
def run(state):
    kind = state["kind"]
    if own:
        return _run_own(state)
    if kind == "tables":
        return _plain_tables(state)
    if kind == "write":
        return _store(state["pool"], state["page"], state["k"], state["v"], state["place"])
    return _plain_attend(state)


def _run_own(s):
    from lit_llama import kv4, pages

    if s["kind"] == "tables":
        r = pages.extend(s["table"], s["seen"], s["free"], s["nfree"], s["slot"], s["add"], s["M"], s["page"], chunk=TABLE_ROWS, commit=False)
        return {"table": s["table"], "row0": r.row0, "row_seq": r.row_seq, "pos": r.pos, "place": r.place, "work": r.work, "seen": r.seen,
                "left": r.left}
    if s["kind"] == "write":
        k, v = s["k"], s["v"]
        layout = kv4.Layout(k.shape[1], k.shape[2], v.shape[2], s["page"])
        kv4.write(s["pool"], layout, k, v, s["place"])
        return kv4.read(s["pool"], layout, s["place"], torch.float32)
    layout = kv4.Layout(s["G"], s["D"], s["D"], s["page"])
    return kv4.attend(s["q"], s["pool"], layout, s["table"], s["slot"], s["pos"], work=None if s["step"] else s["work"], rows=s["per"],
                      sink=s["sink"], gate=s["gate"], count=s["count"])


def _plain_tables(s):
    table, slot, page, M = s["table"], s["slot"].long(), s["page"], s["M"]
    seen, add = s["seen"][slot].long(), s["add"].long()
    have = (seen + page - 1) // page
    new = (seen + add + page - 1) // page - have
    base = torch.cumsum(new, 0) - new
    ends = torch.cumsum(add, 0)
    row0 = torch.cat([torch.zeros_like(ends[:1]), ends])
    m = torch.arange(M, device=DEV)
    b = torch.searchsorted(ends, m, right=True)
    pos = seen[b] + m - row0[b]
    p = pos // page
    at = s["nfree"].long() - 1 - (base[b] + p - have[b])
    fresh = p >= have[b]
    id_ = torch.where(fresh, s["free"][torch.where(fresh, at, torch.zeros_like(at))], table[slot[b], p])
    table[slot[b], p] = id_
    items = (add + TABLE_ROWS - 1) // TABLE_ROWS
    last = torch.cumsum(items, 0)
    t = torch.arange(s["nwork"], device=DEV)
    live = t < last[-1]
    c = torch.searchsorted(last, t, right=True).clamp(max=add.numel() - 1)
    j = (t - (last - items)[c]) * TABLE_ROWS
    work = torch.stack([row0[c] + j, torch.minimum(add[c] - j, torch.full_like(j, TABLE_ROWS)), c], 1)
    work = torch.where(live[:, None], work, torch.zeros_like(work))
    i = torch.int32
    return {"table": table, "row0": row0.to(i), "row_seq": b.to(i), "pos": pos.to(i), "place": (id_ * page + pos % page).to(i), "work": work.to(i),
            "seen": (seen + add).to(i), "left": (s["nfree"] - new.sum()).to(i)}


def _floor_bf16(x):
    """The largest bf16 up to x (float32)."""
    near = x.bfloat16()
    bits = near.view(torch.int16).int()
    down = torch.where(bits == 0, -32767, torch.where(bits < 0, bits + 1, bits - 1)).to(torch.int16).view(torch.bfloat16)
    return torch.where(near.float() > x, down, near)


def _quantize(x):
    """Codes, scale and offset of the vectors x; the quotient in double precision, for codes on a border."""
    x = x.float()
    o = _floor_bf16(x.amin(-1))
    span = x.amax(-1).double() - o.double()
    s = (span / 15).float().bfloat16()
    t = (x.double() - o.double()[..., None]) / torch.where(s == 0, torch.ones_like(s), s).double()[..., None]
    c = torch.where((s == 0)[..., None], torch.zeros_like(t), torch.round(t).clamp(0, 15))
    return c, s, o


def _store(pool, page, k, v, place):
    """k, v (M, G, n) into the pool; what they stand for there."""
    kc, vc, ks, vs = _views(pool, page, k.shape[-1], v.shape[-1])
    p, off = place.long() // page, place.long() % page
    out = []
    for x, codes, pairs in ((k, kc, ks), (v, vc, vs)):
        c, s, o = _quantize(x)
        whole = torch.nn.functional.pad(c.to(torch.uint8), (0, 2 * codes.shape[-1] - c.shape[-1]))
        codes[p, :, off] = whole[..., 0::2] | (whole[..., 1::2] << 4)
        pairs[p, :, off] = torch.stack([s, o], -1)
        out.append(c.float() * s.float()[..., None] + o.float()[..., None])
    return tuple(out)


def _load(codes, pairs, p, off, n):
    """The vectors at pages p, places off, in float32."""
    c = codes[p, :, off]
    c = torch.stack([c & 15, c >> 4], -1).flatten(-2)[..., :n].float()
    so = pairs[p, :, off].float()
    return c * so[..., :1] + so[..., 1:]


def _plain_attend(s):
    page, H, G, D = s["page"], s["H"], s["G"], s["D"]
    table, slot, T, R = s["table"], s["slot"].long(), s["rows"], s["H"] // s["G"]
    B = slot.numel()
    kc, vc, ks, vs = _views(s["pool"], page, D, D)
    j = torch.arange(s["keys"], device=DEV)
    p, off = table[slot[:, None], j // page].long().clamp(min=0), (j % page).expand(B, -1)
    k, v = _load(kc, ks, p, off, D), _load(vc, vs, p, off, D)  # (B, L, G, D)
    pos, b = s["pos"].long(), s["row_seq"].long()
    first = torch.searchsorted(s["row_seq"], torch.arange(B, device=DEV, dtype=torch.int32))
    t = torch.arange(b.numel(), device=DEV) - first[b]
    q = torch.zeros(B, T, H, D, device=DEV)
    q[b, t] = s["q"].float().view(-1, H, D)
    at = torch.full((B, T), -1, device=DEV)
    at[b, t] = pos
    q = q.view(B, T, G, R, D).permute(0, 2, 1, 3, 4).reshape(B, G, T * R, D)
    a = torch.matmul(q, k.permute(0, 2, 3, 1)) * D ** -0.5
    a = a.view(B, G, T, R, -1).masked_fill_(~(j <= at[..., None])[:, None, :, None], -math.inf)
    top = a.amax(-1, keepdim=True)
    top = top.clamp(min=0.0) if s["sink"] else torch.where(top == -math.inf, torch.zeros_like(top), top)
    a = a.sub_(top).exp_()
    total = a.sum(-1, keepdim=True) + (torch.exp(-top) if s["sink"] else 0.0)
    y = torch.matmul(a.view(B, G, T * R, -1), v.permute(0, 2, 1, 3)).view(B, G, T, R, D)
    y = torch.where(total > 0, y / total, torch.zeros_like(y)).permute(0, 2, 1, 3, 4).reshape(B, T, H, D)[b, t]
    if s["gate"] is not None:
        y = y / (1.0 + torch.exp(-s["gate"].float()))[..., None]
    return y.reshape(-1, H * D).to(s["q"].dtype)


# ------------------------------------------------------------------------------------------- what cannot be done without
def work(case) -> dict:
    kind, page = case["kind"], case["page"]
    if kind == "tables":
        adds = _adds(case)
        B, M = case["batch"], sum(adds)
        pages = sum(-(-a // page) for a in adds)
        return {"bytes": 4 * (5 * B + 3 * M + 2 * pages + 3 * (M // TABLE_ROWS + B)), "flops": 8 * M + 8 * B}
    G, D = case["kv_heads"], case["dim"]
    e = 2 if case["dtype"] == "bf16" else 4
    if kind == "write":  # rows in, codes out and in again, values out
        n = case["rows"] * G
        V = case["vdim"]
        return {"bytes": n * ((D + V) * (e + 4) + 2 * ((D + V) / 2 + 8)) + 8 * case["rows"], "flops": 8 * n * (D + V)}
    tokens, rows = _lengths(case)
    H, M = case["heads"], sum(rows)
    pairs = sum(r * t - r * (r - 1) // 2 for t, r in zip(tokens, rows) if t)
    return {"bytes": sum(tokens) * G * (D + 8) + M * H * D * 2 * e + (M * H * e if case["gate"] else 0) + 4 * sum(-(-t // page) for t in tokens) + 8 * M,
            "flops": 4 * D * H * pairs}


# ------------------------------------------------------------------------------------------- in double precision
def exact(case, seed):
    """The definition, sequence by sequence and head by head, in 64 bits."""
    s = prepare(case, seed)
    if s["kind"] == "tables":
        return _exact_tables(s)
    if s["kind"] == "write":
        return tuple(_stands_for(s[n].double()) for n in ("k", "v"))
    page, H, G, D = s["page"], s["H"], s["G"], s["D"]
    R, kb = H // G, s["page"] * _width(s["D"]) // 2
    y = torch.zeros(s["pos"].numel(), H, D, dtype=torch.float64, device=DEV)
    q = s["q"].double().view(-1, H, D)
    row = 0
    for b, (L, n) in enumerate(zip(s["tokens"], s["new"])):
        if L:
            blocks = s["pool"][s["table"][b, :-(-L // page)].long()]  # (pages, G, bytes)
            visible = torch.arange(L, device=DEV)[None] <= torch.arange(L - n, L, device=DEV)[:, None]
            for g in range(G):
                k = _decode(blocks[:, g, :kb], blocks[:, g, 2 * kb:2 * kb + 4 * page], page, D)[:L]
                v = _decode(blocks[:, g, kb:2 * kb], blocks[:, g, 2 * kb + 4 * page:], page, D)[:L]
                for h in range(g * R, (g + 1) * R):
                    e = (q[row:row + n, h] @ k.T) / math.sqrt(D)
                    e = torch.where(visible, e, torch.full_like(e, -math.inf))
                    if s["sink"]:
                        e = torch.cat([e, torch.zeros_like(e[:, :1])], 1)
                    y[row:row + n, h] = torch.softmax(e, 1)[:, :L] @ v
        row += n
    if s["gate"] is not None:
        y *= torch.sigmoid(s["gate"].double())[..., None]
    return y.view(-1, H * D)


def _exact_tables(s) -> dict:
    """Request by request on the host."""
    page, table, free, seen = s["page"], s["table"].tolist(), s["free"].tolist()[:int(s["nfree"])], s["seen"].tolist()
    out = {"row0": [0], "row_seq": [], "pos": [], "place": [], "work": [], "seen": []}
    for b, (x, n) in enumerate(zip(s["slot"].tolist(), s["add"].tolist())):
        out["work"] += [[len(out["pos"]) + j, min(TABLE_ROWS, n - j), b] for j in range(0, n, TABLE_ROWS)]
        held = -(-seen[x] // page)
        for t in range(seen[x], seen[x] + n):
            if t // page >= held:
                table[x][held] = free.pop()
                held += 1
            out["pos"].append(t)
            out["row_seq"].append(b)
            out["place"].append(table[x][t // page] * page + t % page)
        out["seen"].append(seen[x] + n)
        out["row0"].append(len(out["pos"]))
    out["work"] += [[0, 0, 0]] * (s["nwork"] - len(out["work"]))
    out.update(table=table, left=[len(free)])
    return {k: torch.tensor(v, dtype=torch.int32) for k, v in out.items()}


def _decode(codes, pairs, page, n):
    """A head's vectors out of its bytes in every page, (pages page, n)."""
    c = codes.reshape(codes.shape[0] * page, -1)
    so = pairs.contiguous().view(torch.bfloat16).view(-1, 2).double()
    w = torch.empty(c.shape[0], 2 * c.shape[1], dtype=torch.float64, device=DEV)
    w[:, 0::2], w[:, 1::2] = c % 16, c // 16
    return w[:, :n] * so[:, :1] + so[:, 1:]


def _stands_for(x):
    lo, hi = x.min(-1).values, x.max(-1).values
    ulp = torch.exp2(torch.floor(torch.log2(lo.abs().clamp(min=1e-30))) - 7)  # of a bf16 of that size
    o = torch.floor(lo / ulp) * ulp
    s = ((hi - o) / 15.0).float().to(torch.bfloat16).double()
    c = torch.clamp(torch.round((x - o[..., None]) / s[..., None]), 0, 15)
    return c * s[..., None] + o[..., None]
