"""The cache's operators together, as a model's decode steps use them: prompt,
steps, eviction; captured into a CUDA graph; on several streams at once."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kv_reference as ref
from test_gpu_kv import make, queries

pytestmark = pytest.mark.gpu


def small(layers, bposit=False):
    from bposit_b200.forward import QWEN05, QwenShaped
    from bposit_b200.nn import bpositify
    m = QwenShaped(dict(QWEN05, vocab=500), layers=layers).cuda().init_weights(1)
    return bpositify(m) if bposit else m


@pytest.mark.parametrize("fmt", ["bp8", "bp16"])
def test_prefill_is_the_forward_and_fills_the_cache(orc, fmt):
    m = small(2)
    g = torch.Generator(device="cuda").manual_seed(0)
    ids = torch.randint(0, 500, (3, 37), generator=g, device="cuda")
    seen = []
    cos, sin = (torch.cat((t, t), -1)[None, None] for t in m.rope_tables(37))
    m.layers[0](m.embed(ids), cos, sin, store=lambda k, v: seen.append((k.detach().cpu(), v.detach().cpu())))
    lengths = [37, 5, 20]
    cache = m.new_cache(3, 50, fmt, page_size=16, track=True)
    untouched = cache.k.clone()
    assert torch.equal(m.prefill(ids, cache, lengths), m(ids))
    assert cache.lengths.tolist() == lengths and cache.seen.tolist() == lengths and cache.longest == 37
    k, v = seen[0]
    table = cache.page_table.cpu().numpy()
    for b, n in enumerate(lengths):
        at = np.arange(n)
        for x, pool, exps in ((k, cache.k, cache.k_exp), (v, cache.v, cache.v_exp)):
            codes, e = ref.encode(orc, x[b, :, :n].transpose(0, 1).contiguous(), fmt)
            got = pool.cpu().numpy()[0][table[b, at // 16], :, at % 16]
            assert np.array_equal(got, codes)
            if e is not None:
                assert np.array_equal(exps.cpu().numpy()[0][table[b, at // 16], :, at % 16], e)
        assert torch.equal(cache.positions[0, b, 1, :n].cpu(), torch.arange(n, dtype=torch.int32))
        page = int(table[b, 3])        # nothing behind the length
        assert torch.equal(cache.k[:, page].view(torch.uint8), untouched[:, page].view(torch.uint8))
    with pytest.raises(ValueError, match="empty"):
        m.prefill(ids, cache)


@pytest.mark.parametrize("fmt", ["bp8", "bp16"])
def test_step_matches_plain_attention_over_the_cache(orc, fmt, monkeypatch):
    """One layer, so that nothing is encoded behind the attention.  Against the same step with 64-bit attention: both
    are sums of at most 4864 fp32 products of the hidden state's magnitude, 4864 half steps of 2^-24 each."""
    from bposit_b200 import ops
    m = small(1)
    g = torch.Generator(device="cuda").manual_seed(3)
    ids = torch.randint(0, 500, (4, 33), generator=g, device="cuda")
    token = torch.randint(0, 500, (4,), generator=g, device="cuda")
    tables = m.rope_tables(64)
    got = []
    for plain in (False, True):
        cache = m.new_cache(4, 40, fmt, page_size=16)
        m.prefill(ids, cache, [33, 1, 16, 20])
        if plain:
            tab = ref.code_values(orc, fmt)
            monkeypatch.setattr(ops, "paged_attention", lambda c, q, layer=0, **kw:
                                ref.attention(c, tab, q, layer)[0].float().cuda())
        got.append(m.step(token, cache, tables))
        assert cache.lengths.tolist() == [34, 2, 17, 21]
    scale = got[1].abs().max()
    assert (got[0] - got[1]).abs().max() <= 4864 * 2.0 ** -24 * scale


def test_generate_with_and_without_a_budget():
    m = small(2, bposit=True)
    g = torch.Generator(device="cuda").manual_seed(5)
    ids = torch.randint(0, 500, (3, 40), generator=g, device="cuda")
    all_of_it = m.generate(ids, 6, page_size=16)
    assert all_of_it.shape == (3, 6) and all_of_it.dtype == torch.int64
    assert torch.equal(m.generate(ids, 6, page_size=16), all_of_it)
    # a budget that is never reached changes nothing
    assert torch.equal(m.generate(ids, 6, page_size=16, budget=64), all_of_it)
    assert m.generate(ids, 30, page_size=16, budget=24, recent=8, sinks=2).shape == (3, 30)
    assert torch.equal(m.generate(ids, 6, lengths=[40, 40, 40], page_size=16), all_of_it)
    for kw in (dict(new_tokens=0), dict(new_tokens=2, lengths=[3, 0, 1]), dict(new_tokens=2, budget=0)):
        with pytest.raises(ValueError):
            m.generate(ids, **kw)


@pytest.mark.parametrize("track", [False, True])
def test_a_captured_step_goes_on_with_every_replay(track):
    m = small(2)
    g = torch.Generator(device="cuda").manual_seed(6)
    ids = torch.randint(0, 500, (2, 30), generator=g, device="cuda")
    tokens = torch.randint(0, 500, (6, 2), generator=g, device="cuda")
    tables = m.rope_tables(64)
    caches = [m.new_cache(2, 40, page_size=16, track=track) for _ in range(2)]
    for c in caches:
        m.prefill(ids, c, [30, 17])
    want = [m.step(t, caches[0], tables) for t in tokens]
    token = tokens[0].clone()
    got = [m.step(token, caches[1], tables)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.step(token, caches[1], tables)
    for t in tokens[1:5]:
        token.copy_(t)
        graph.replay()
        got.append(out.clone())
    assert caches[1].longest == 32 and caches[1].bound is None and caches[0].bound == 36
    got.append(m.step(tokens[5], caches[1], tables))      # and without the graph again
    # the entries are the same; the split of the sums does not depend on max_length
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert caches[1].lengths.tolist() == [36, 23] and torch.equal(caches[0].k, caches[1].k)
    if track:
        assert torch.equal(caches[0].scores, caches[1].scores)
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            caches[0].evict(5)                            # captured, not run: the host still knows the lengths
        assert caches[0].longest == 36 and caches[0].bound is None


def test_steps_and_evictions_keep_what_they_promise():
    m = small(2)
    g = torch.Generator(device="cuda").manual_seed(7)
    ids = torch.randint(0, 500, (2, 50), generator=g, device="cuda")
    cache = m.new_cache(2, 64, "bp8", page_size=16, track=True)
    tables = m.rope_tables(200)
    m.prefill(ids, cache, [50, 30])
    for n in range(1, 60):
        m.step(torch.randint(0, 500, (2,), generator=g, device="cuda"), cache, tables)
        if cache.longest > 56:
            cache.evict(40, recent=10, sinks=3)
            held = cache.lengths.tolist()
            assert cache.longest == 40 and max(held) <= 40
            for b, first in enumerate((50, 30)):
                for layer in range(2):
                    for hk in range(2):
                        pos = cache.positions[layer, b, hk, : held[b]].tolist()
                        assert len(set(pos)) == held[b]
                        assert {0, 1, 2} <= set(pos) and set(range(first + n - 10, first + n)) <= set(pos)
    assert cache.seen.tolist() == [50 + 59, 30 + 59]
    # every weight that was given is somewhere: no entry has more than all tokens of all its heads gave
    assert cache.scores.ge(0).all() and cache.scores.max() <= 7 * 59 * (1 + 1e-5)
    with pytest.raises(ValueError, match="capacity"):
        cache.advance(100)
    cache.reset()
    assert cache.longest == 0 and not cache.lengths.any()


def decode(cache, k, v, q, tables, pos, weights):
    from bposit_b200 import ops
    r = ops.kv_append(cache, k, v, q=q, cos=tables[0], sin=tables[1], positions=pos)
    out = ops.paged_attention(cache, r, accumulate=True)
    keep = ops.kv_evict(cache, 60, recent=4, sinks=1, weights=weights)
    return out, keep


def state(seed):
    cache = make(4, 2, 64, [64, 5, 64, 33], "bp8", 16, track=True, seed=seed)
    x = queries(4, 8, 64, seed=seed + 1)
    k, v, q = x[:, :2], x[:, 2:4], x[:, 4:]
    ang = torch.rand(80, 32, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
    pos = torch.tensor([70, 4, 79, 32], dtype=torch.int32, device="cuda")
    w = torch.rand(cache.scores.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed + 2))
    return cache, k, v, q, (ang.cos(), ang.sin()), pos, w


def contents(cache):
    return [t.clone() for t in (cache.k, cache.v, cache.k_exp, cache.v_exp, cache.positions, cache.scores)]


def test_captured_steps_replay_as_they_ran():
    args = [state(11), state(12)]
    want = []
    for a in args:
        want.append((*decode(*a), *contents(a[0])))
    args = [state(11), state(12)]
    start = [contents(a[0]) for a in args]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for a in args:          # two graphs, replayed at the same time on two streams
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(decode(*a))
        graphs.append(g)
    for _ in range(3):
        for a, s in zip(args, start):
            for t, u in zip((a[0].k, a[0].v, a[0].k_exp, a[0].v_exp, a[0].positions, a[0].scores), s):
                t.copy_(u)
        torch.cuda.synchronize()
        for g in graphs:
            with torch.cuda.stream(torch.cuda.Stream()):
                g.replay()
        torch.cuda.synchronize()
        for a, o, w in zip(args, outs, want):
            assert all(torch.equal(x, y) for x, y in zip((*o, *contents(a[0])), w))


def test_calls_on_several_streams_at_once():
    from bposit_b200 import ops
    caches = [make(3, 2, 64, [2000 + 7 * i, 900, 64], "bp8" if i % 2 else "bp16", 64, track=True, seed=i)
              for i in range(4)]
    qs = [queries(3, 14, 64, seed=20 + i) for i in range(4)]
    want = [ops.paged_attention(c, q) for c, q in zip(caches, qs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = [[] for _ in range(4)]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.paged_attention(caches[i], qs[i]))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, x) for x in g)


def test_own_workspace_and_library_workspace_agree():
    """The C entry with the caller's workspace, and with none."""
    import ctypes

    from bposit_b200 import _lib, ops
    L = _lib.lib()
    cache = make(3, 2, 64, [1500, 3, 700], "bp8", 64, track=True)
    q = queries(3, 14, 64)
    want = ops.paged_attention(cache, q)
    out = torch.empty_like(want)
    for acc in (0, 1):
        rc = L.bp_paged_attention(cache._ref, 0, 0, 14, q.data_ptr(), q.stride(0), out.data_ptr(), None, 0.125, 0, acc,
                                  None, 0, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert rc == 0
        torch.cuda.synchronize()
        assert torch.equal(out, want)
