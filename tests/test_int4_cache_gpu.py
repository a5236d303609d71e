"""Bobasun with its keys and values in 4 bits (new_state(.., cache="int4")): the same model in double precision whose attention reads what
the codes stand for, through prompts, portions, decode steps in a captured graph, unequal batches and slots used again.

The rounding of a key to its code hangs on the last bit of the rotated key, which the model and the oracle form in different precisions: a code that
falls on the other side of a border is one step off, as large as the error that the 4 bits themselves make. So logits are held to a
share of what the 4 bits change: 0.25 of the distance between the oracle with and without them in float32 (where codes hardly ever differ), and the
whole of it, beside the type's own tolerance, in bfloat16 (whose rounding of activations moves codes everywhere)."""
import numpy as np
import pytest
import torch

from oracle import bobasun_np as B
from oracle import kv4_np as O
from tests.bobasun_cases import CONFIGS, build, config, layer, oracle, prompts, weights

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]
NAMES = ["odd", "tiled", "wide"]
_cache = {}


def case(name, dtype):
    if (name, dtype) not in _cache:
        w = weights(CONFIGS[name], 0)
        _cache[name, dtype] = (CONFIGS[name], w, build(CONFIGS[name], w, dtype))
    return _cache[name, dtype]


def through_codes(cfg, w, toks, monkeypatch, dtype):
    """The oracle whose attention reads what keys and values (rounded to the type, as they are written) stand for in 4 bits."""
    real = B.sink_attention

    def coded(q, k, v, scale):
        def code(x):
            x = torch.tensor(np.ascontiguousarray(x)).to(dtype).float().numpy()
            return O.stands_for(x)

        return real(q, code(k), code(v), scale)

    with monkeypatch.context() as m:
        m.setattr(B, "sink_attention", coded)
        return oracle(cfg, w, toks)


def near(got, want, plain, dtype, what=""):
    """Root mean square over the rows: the 4 bits' own effect is `want` against `plain`."""
    got = got.double().cpu().numpy() if isinstance(got, torch.Tensor) else got
    off, own = np.sqrt(((got - want) ** 2).mean()), np.sqrt(((want - plain) ** 2).mean())
    scale = np.abs(plain).max()
    limit = 0.25 * own + 5e-5 * scale if dtype == torch.float32 else own + 0.02 * scale
    assert np.isfinite(got).all() and off < limit, f"{what}: {off:.3g}, the 4 bits' own {own:.3g}, limit {limit:.3g}"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", NAMES)
def test_prompts_and_portions(hip, monkeypatch, name, dtype):
    cfg, w, m = case(name, dtype)
    for n in (1, 17, 64, 65, 200):
        toks = prompts(cfg, [n], seed=n)[0]
        want, plain = through_codes(cfg, w, toks, monkeypatch, dtype), oracle(cfg, w, toks)
        st = m.new_state(1, cache="int4")
        near(m.extend(st, st.alloc(1), [0], [toks]), want, plain, dtype, (name, n))
        st.check()
    st = m.new_state(2, cache="int4")
    slot = st.alloc(1)
    got = [m.extend(st, slot, [p], [toks[p:p + 37]]) for p in range(0, len(toks), 37)]
    near(torch.cat(got), want, plain, dtype, "portions")
    st.check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", NAMES)
def test_decode_steps_equal_the_prompt(hip, monkeypatch, name, dtype):
    """Token by token through the session's graph, past pages and grown pools."""
    from lit_llama.engine import DecodeSession

    cfg, w, m = case(name, dtype)
    toks = prompts(cfg, [150], seed=2)[0]
    want, plain = through_codes(cfg, w, toks, monkeypatch, dtype), oracle(cfg, w, toks)
    s = DecodeSession(m, 1, None, None, keep_tokens=False, state=m.new_state(1, cache="int4"))
    out = [s.prefill([toks[:1]], want=[[0]]).clone()]
    for t in toks[1:]:
        out.append(s.feed([t]).clone())
    near(torch.cat(out), want, plain, dtype)
    s.check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_unequal_batch_early_ends_and_slots_again(hip, monkeypatch, dtype):
    from lit_llama.engine import DecodeSession

    cfg, w, m = case("tiled", dtype)
    state = m.new_state(4, cache="int4")
    for turn in range(2):
        lens, extra = ([1, 150, 37, 70], [3, 9, 6, 9]) if turn == 0 else ([66, 2, 129], [5, 12, 1])
        toks = prompts(cfg, [a + b for a, b in zip(lens, extra)], seed=10 + turn)
        refs = [(through_codes(cfg, w, t, monkeypatch, dtype), oracle(cfg, w, t)) for t in toks]
        s = DecodeSession(m, len(lens), None, None, state=state, keep_tokens=False)
        s.prefill([t[:n] for t, n in zip(toks, lens)])
        live, at, got, want, plain = list(range(len(lens))), list(lens), [], [], []
        while live:
            got.append(s.feed([toks[i][at[i]] for i in live]).clone())
            want += [refs[i][0][at[i]] for i in live]
            plain += [refs[i][1][at[i]] for i in live]
            for i in live:
                at[i] += 1
            done = [k for k, i in enumerate(live) if at[i] == len(toks[i])]
            if done:
                s.check()
                s.finish(done)
                live = [i for k, i in enumerate(live) if k not in done]
        near(torch.cat(got), np.stack(want), np.stack(plain), dtype)
        assert len(state._free) == 4 and int(state.nfree) == state.free.numel() and not state.seen.any()


def test_generate_and_memory(hip):
    """generate() with the option; the cache takes less than 0.3 of the bf16 rows at heads of 128; same tokens from the graph and without."""
    from lit_llama.engine import DecodeSession
    import generate as G

    cfg = config(256, 128, 2, [layer(8, 2, 128, 128, 256) for _ in range(2)])
    m = build(cfg, weights(cfg, 3), torch.bfloat16)
    idx = torch.tensor(prompts(cfg, [40], seed=4)[0], device="cuda")
    y = G.generate(m, idx, 30, top_k=1, kv_cache="int4")
    assert y.shape == (70,) and torch.equal(y[:40], idx)
    s = DecodeSession(m, 1, 70, 70, use_graph=False, state=m.new_state(1, 70, "int4"))
    s.prefill(idx.view(1, -1))
    s.decode(29)
    s.check()
    assert torch.equal(s.output()[0].to(idx.dtype), y)
    four, full = m.new_state(1, cache="int4"), m.new_state(1, 4096)
    four.room(four.alloc(1), [4096])
    assert sum(p.numel() for p in four.pool.values()) < 0.3 * sum(2 * r.numel() for r in full.ring.values())


def test_rows_that_begin_elsewhere(hip):
    """A call goes on where its sequences end: one that begins before or behind that, or names a slot twice, raises."""
    cfg, w, m = case("tiled", torch.bfloat16)
    for starts, again in (([3], [0]), ([9], [0]), ([5, 5], [0, 0])):
        st = m.new_state(2, cache="int4")
        slot = st.alloc(1)
        m.extend(st, slot, [0], [[1, 2, 3, 4, 5]])
        with pytest.raises(RuntimeError, match="not valid"):
            m.extend(st, [slot[k] for k in again], starts, [[1, 2]] * len(starts))


def test_what_is_refused(hip):
    from lit_llama import LLaMA, LLaMAConfig
    import generate as G

    cfg, w, m = case("tiled", torch.bfloat16)
    with pytest.raises(ValueError):
        m.new_state(1, cache="int8")
    st = m.new_state(2, 50, "int4")
    slots = st.alloc(2)
    with pytest.raises(ValueError):
        st.room(slots, [51, 3])
    with pytest.raises(ValueError):
        st.release([slots[0], slots[0]])
    st.release(slots)
    with pytest.raises(ValueError):
        st.release([slots[0]])
    big = build(config(64, 32, 1, [layer(1, 1, 264, 8, None)]), weights(config(64, 32, 1, [layer(1, 1, 264, 8, None)])), torch.bfloat16)
    with pytest.raises(ValueError):
        big.new_state(1, cache="int4")
    with pytest.raises(ValueError):
        G.generate(LLaMA(LLaMAConfig(block_size=8, vocab_size=32, n_layer=1, n_head=1, n_embd=64)), torch.zeros(2, dtype=torch.long), 2, kv_cache="int4")
