"""The paged b-posit key-value cache on the GPU against plain 64-bit forms:
appending rotated tokens, attention of one token per sequence, eviction by
accumulated weight, and the three together in a model."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import kv_reference as ref

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make(batch, kv_heads, dim, lengths, fmt="bp8", page=16, layers=1, track=False, seed=0, spare=2, per=None,
         fill="normal"):
    """A cache over a shuffled pool whose every row is filled, held or not."""
    from bposit_b200.kv import PagedKVCache
    g = torch.Generator(device="cuda").manual_seed(seed)
    per = max(1, -(-max(lengths) // page)) if per is None else per
    pages = batch * per + spare
    shape = (layers, pages, kv_heads, page)
    n = math.prod(shape) * dim
    if fmt == "bp8":
        k, v = (torch.randint(0, 256, (n,), generator=g, device="cuda").to(torch.uint8) for _ in range(2))
        if fill == "normal":      # magnitudes 2^-5 .. 2^5, as rows around 1 have them
            k, v = (torch.where(x < 128, 24 + x % 80, 256 - (24 + x % 80)).to(torch.uint8) for x in (k.int(), v.int()))
        ke, ve = (torch.randint(-4, 2, shape, generator=g, device="cuda", dtype=torch.int8) for _ in range(2))
    else:
        k, v = (torch.randint(-32768, 32768, (n,), generator=g, device="cuda") for _ in range(2))
        if fill == "normal":
            k, v = (torch.where(x >= 0, 12000 + x % 7000, -(12000 + x % 7000)) for x in (k, v))
        k, v = (x.to(torch.int16).view(torch.uint16) for x in (k, v))
        ke = ve = None
    table = torch.randperm(pages, generator=g, device="cuda")[: batch * per].view(batch, per).to(torch.int32)
    pos = scores = None
    if track:
        pos = torch.arange(per * page, device="cuda", dtype=torch.int32).expand(layers, batch, kv_heads, -1).contiguous()
        scores = torch.rand(pos.shape, generator=g, device="cuda")
    return PagedKVCache.over(k.view(shape + (dim,)), v.view(shape + (dim,)), table,
                             torch.tensor(lengths, dtype=torch.int32, device="cuda"), k_exp=ke, v_exp=ve,
                             positions=pos, scores=scores)


def queries(batch, heads, dim, dtype=torch.float32, seed=1, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(batch, heads, dim, generator=g, device="cuda") * size).to(dtype)


def check_attention(orc, cache, q, layer=0, scale=None, **kw):
    from bposit_b200 import ops
    tab = ref.code_values(orc, cache.fmt)
    want, lse_want, weights, bound, lse_bound = ref.attention(cache, tab, q, layer, scale)
    got, lse = ops.paged_attention(cache, q, layer=layer, scale=scale, return_lse=True, **kw)
    got, lse = got.double().cpu(), lse.double().cpu()
    tol = bound + HALF_STEP[q.dtype] * 1.01 * (want.abs() + bound) + (2.0 ** -25 if q.dtype == torch.float16 else 0)
    bad = (got - want).abs() > tol
    assert not bad.any(), (bad.sum().item(), ((got - want).abs() / tol).max().item())
    none = torch.isinf(lse_want)
    assert torch.equal(torch.isinf(lse), none) and (lse[~none] - lse_want[~none]).abs().le(lse_bound[~none]).all()
    return weights


LENGTHS = [[0, 1, 2, 15, 16, 17, 31], [63, 64, 65, 0, 127, 129, 1], [1000, 3, 517], [2311]]


@pytest.mark.parametrize("fmt", ["bp8", "bp16"])
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("heads,kv_heads,page,which", [(14, 2, 64, 0), (9, 3, 16, 1), (4, 4, 32, 2), (16, 1, 128, 3)])
def test_attention_matches_64_bits(orc, fmt, dim, heads, kv_heads, page, which):
    lens = LENGTHS[which]
    cache = make(len(lens), kv_heads, dim, lens, fmt, page, seed=dim + which)
    check_attention(orc, cache, queries(len(lens), heads, dim))


@pytest.mark.parametrize("fmt", ["bp8", "bp16"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_16_bit_activations(orc, fmt, dtype):
    lens = [1, 70, 333, 0]
    cache = make(4, 2, 64, lens, fmt, 32)
    check_attention(orc, cache, queries(4, 6, 64, dtype))


@pytest.mark.parametrize("fmt", ["bp8", "bp16"])
def test_attention_of_every_code(orc, fmt):
    """Random codes of all values (zero and NaR among them): tiny queries keep the scores apart from one-hot."""
    lens = [200, 77]
    cache = make(2, 2, 64, lens, fmt, 16, fill="all")
    check_attention(orc, cache, queries(2, 4, 64, size=2.0 ** (-26 if fmt == "bp8" else -114)))


def test_attention_wide_exponents(orc):
    """Row exponents over int8's range: keys scaled down to nothing, values from 2^-128 to 2^100."""
    cache = make(3, 1, 64, [50, 64, 9], "bp8", 16)
    g = torch.Generator(device="cuda").manual_seed(3)
    cache.k_exp.copy_(torch.randint(-128, -10, cache.k_exp.shape, generator=g, device="cuda"))
    for lo, hi in ((-128, -90), (60, 101), (-20, 20)):
        cache.v_exp.copy_(torch.randint(lo, hi, cache.v_exp.shape, generator=g, device="cuda"))
        check_attention(orc, cache, queries(3, 4, 64))


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3])
def test_attention_scale(orc, scale):
    cache = make(2, 2, 32, [40, 100], "bp8", 16)
    check_attention(orc, cache, queries(2, 4, 32), scale=scale)


def test_large_scores_stay_finite(orc):
    """Scores of thousands: the running maximum keeps every exponential in range."""
    cache = make(2, 1, 64, [300, 64], "bp16", 16)
    check_attention(orc, cache, queries(2, 8, 64, size=300.0))


@pytest.mark.parametrize("fmt", ["bp8", "bp16"])
def test_rows_behind_the_length_are_never_used(orc, fmt):
    from bposit_b200 import ops
    lens = [5, 16, 100, 0]
    cache = make(4, 2, 64, lens, fmt, 16, per=8)
    q = queries(4, 6, 64)
    before = ops.paged_attention(cache, q)
    for b, n in enumerate(lens):
        for i in range(n, cache.capacity):
            page = int(cache.page_table[b, i // 16])
            for pool in (cache.k, cache.v):
                (pool if fmt == "bp8" else pool.view(torch.int16))[0, page, :, i % 16] = 0x80 if fmt == "bp8" else -32768
            if fmt == "bp8":
                cache.k_exp[0, page, :, i % 16] = 127
                cache.v_exp[0, page, :, i % 16] = 127
    assert torch.equal(ops.paged_attention(cache, q), before)
    # pages past the length are not even looked up
    for b, n in enumerate(lens):
        cache.page_table[b, -(-n // 16):] = -7
    assert torch.equal(ops.paged_attention(cache, q), before)


def test_lengths_are_cut_to_the_capacity_and_max_length(orc):
    from bposit_b200 import ops
    cache = make(3, 2, 64, [64, 64, 20], "bp8", 16)
    q = queries(3, 4, 64)
    cut = ops.paged_attention(cache, q, max_length=23)
    # (compared at equal effective lengths: the order of a sum depends on how the whole batch is split)
    cache.lengths.copy_(torch.tensor([64, 64, 0]))
    full = ops.paged_attention(cache, q)
    cache.lengths.copy_(torch.tensor([1 << 30, 64, -5]))
    got = ops.paged_attention(cache, q)
    assert torch.equal(got, full) and full[:2].any() and not got[2].any()
    cache.lengths.copy_(torch.tensor([23, 23, 20]))
    assert torch.equal(ops.paged_attention(cache, q), cut)


def test_a_page_outside_the_pool_gives_nan_for_its_sequence_only(orc):
    from bposit_b200 import ops
    for bad in (-1, 1 << 30, -(1 << 31)):
        cache = make(3, 2, 64, [70, 200, 33], "bp8", 16, track=True)
        q = queries(3, 4, 64)
        good = ops.paged_attention(cache, q)
        cache.scores.zero_()
        cache.page_table[1, 7] = bad
        got, lse = ops.paged_attention(cache, q, accumulate=True, return_lse=True)
        assert torch.equal(got[0], good[0]) and torch.equal(got[2], good[2])
        assert got[1].isnan().all() and lse[1].isnan().all()
        assert not cache.scores[0, 1].any() and cache.scores[0, 0, :, :70].gt(0).all()


def test_non_finite_queries_give_nan_and_touch_no_other_head(orc):
    from bposit_b200 import ops
    cache = make(2, 2, 64, [90, 20], "bp8", 16)
    q = queries(2, 8, 64)
    good = ops.paged_attention(cache, q)
    q[0, 1, 5], q[1, 6, 0] = float("nan"), float("inf")
    got = ops.paged_attention(cache, q)
    hit = torch.zeros(2, 8, dtype=torch.bool, device="cuda")
    hit[0, 1] = hit[1, 6] = True
    assert got[hit].isnan().all() and torch.equal(got[~hit], good[~hit])


@pytest.mark.parametrize("length", [20, 3000])
def test_scores_behind_a_page_outside_the_pool_stay(orc, length):
    from bposit_b200 import ops
    cache = make(2, 2, 64, [length, 50], "bp8", 16, track=True)
    q = queries(2, 8, 64)
    good, start = ops.paged_attention(cache, q), cache.scores.clone()
    cache.page_table[0, 0] = cache.pages
    got = ops.paged_attention(cache, q, accumulate=True)
    assert torch.equal(cache.scores[0, 0], start[0, 0]) and got[0].isnan().all() and torch.equal(got[1], good[1])
    assert cache.scores[0, 1, :, :50].gt(start[0, 1, :, :50]).any() and cache.scores.isfinite().all()


@pytest.mark.parametrize("length", [20, 3000])
def test_scores_of_a_kv_head_with_a_nan_query_stay(orc, length):
    from bposit_b200 import ops
    cache = make(2, 2, 64, [length, 50], "bp8", 16, track=True)
    q = queries(2, 8, 64)
    q[0, 6, 1] = float("nan")                       # kv head 1 of sequence 0
    start = cache.scores.clone()
    ops.paged_attention(cache, q, accumulate=True)
    assert torch.equal(cache.scores[0, 0, 1], start[0, 0, 1])
    assert cache.scores[0, 0, 0, :length].gt(start[0, 0, 0, :length]).any()
    assert cache.scores[0, 1, :, :50].gt(start[0, 1, :, :50]).any() and cache.scores.isfinite().all()


@pytest.mark.parametrize("fmt,heads,kv_heads,dim", [("bp8", 9, 3, 64), ("bp16", 4, 4, 32), ("bp8", 20, 2, 128)])
def test_accumulated_weights(orc, fmt, heads, kv_heads, dim):
    from bposit_b200 import ops
    lens = [0, 1, 150, 64, 399]
    cache = make(5, kv_heads, dim, lens, fmt, 16, layers=2, track=True)
    q = queries(5, heads, dim)
    start = cache.scores.clone()
    weights = check_attention(orc, cache, q, layer=1, accumulate=True)
    assert torch.equal(cache.scores[0], start[0])
    for b, n in enumerate(lens):
        for hk in range(kv_heads):
            got, was = cache.scores[1, b, hk].double().cpu(), start[1, b, hk].double().cpu()
            assert torch.equal(got[n:], was[n:])
            if n:
                want = was[:n] + weights[b, hk]
                # the sum over the heads and onto the score: one half step each
                tol = weights[b, hk, "bound"] + (heads // kv_heads + 1) * 2.0 ** -24 * want.abs()
                assert (got[:n] - want).abs().le(tol).all()


@pytest.mark.parametrize("fmt,heads,kv_heads,dim,dtype", [
    ("bp8", 14, 2, 64, torch.float32), ("bp8", 3, 3, 96, torch.bfloat16), ("bp16", 12, 1, 128, torch.float32),
    ("bp16", 8, 4, 32, torch.float16), ("bp8", 17, 1, 32, torch.float32), ("bp16", 2, 2, 96, torch.float32)])
def test_accumulated_weights_of_long_rows(orc, fmt, heads, kv_heads, dim, dtype):
    """Rows that are split over several blocks, one that is not, and an empty one."""
    lens = [5003, 0, 777, 31]
    cache = make(4, kv_heads, dim, lens, fmt, 64, track=True)
    start = cache.scores.clone()
    weights = check_attention(orc, cache, queries(4, heads, dim, dtype), accumulate=True)
    for b, n in enumerate(lens):
        for hk in range(kv_heads):
            got, was = cache.scores[0, b, hk].double().cpu(), start[0, b, hk].double().cpu()
            assert torch.equal(got[n:], was[n:])
            if n:
                want = was[:n] + weights[b, hk]
                tol = weights[b, hk, "bound"] + (heads // kv_heads + 1) * 2.0 ** -24 * want.abs()
                assert (got[:n] - want).abs().le(tol).all()


def test_attention_results_repeat_bit_for_bit(orc):
    from bposit_b200 import ops
    cache = make(6, 2, 64, [2000, 3, 700, 0, 64, 1234], "bp8", 64, track=True)
    q = queries(6, 14, 64)
    first, start = ops.paged_attention(cache, q, accumulate=True), cache.scores.clone()
    for _ in range(3):
        assert torch.equal(ops.paged_attention(cache, q), first)
    cache.scores.copy_(start)
    a = ops.paged_attention(cache, q, accumulate=True), cache.scores.clone()
    cache.scores.copy_(start)
    b = ops.paged_attention(cache, q, accumulate=True), cache.scores.clone()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_results_may_replace_the_queries(orc, dtype):
    from bposit_b200 import ops
    cache = make(3, 2, 64, [4000, 5, 0], "bp8", 64)
    q = queries(3, 14, 64, dtype)
    want = ops.paged_attention(cache, q)
    mine = q.clone()
    assert ops.paged_attention(cache, mine, out=mine) is mine and torch.equal(mine, want)
    for tokens in (3, 2600):
        x = queries(tokens, 14, 64, dtype, seed=3)
        k = queries(tokens, 2, 64, dtype, seed=4)
        cos = torch.rand(4000, 32, device="cuda")
        at = torch.arange(tokens, device="cuda", dtype=torch.int32)
        args = dict(cos=cos, sin=1 - cos, seqs=torch.zeros_like(at), places=at)
        want = ops.kv_append(cache, k, k, q=x, **args)
        mine = x.clone()
        assert ops.kv_append(cache, k, k, q=mine, q_out=mine, **args) is mine and torch.equal(mine, want)


def test_calls_with_nothing_to_do(orc):
    from bposit_b200 import ops
    cache = make(3, 2, 64, [0, 0, 0], "bp8", 16, track=True, per=2)
    out, lse = ops.paged_attention(cache, queries(3, 4, 64), accumulate=True, return_lse=True)
    assert not out.any() and lse.eq(-math.inf).all()
    was = cache.k.clone(), cache.scores.clone()
    none = torch.zeros(0, device="cuda", dtype=torch.int32)
    cos = torch.rand(8, 32, device="cuda")
    q = ops.kv_append(cache, queries(0, 2, 64), queries(0, 2, 64), q=queries(0, 4, 64), cos=cos, sin=cos, seqs=none,
                      places=none)
    assert q.shape == (0, 4, 64)
    assert ops.kv_evict(cache, 3).eq(-1).all()
    assert torch.equal(cache.k, was[0]) and torch.equal(cache.scores, was[1])


def test_calls_on_two_streams_at_once_and_in_one_graph(orc):
    """Two caches whose calls run beside each other, eagerly, from two threads, and as branches of a graph."""
    import threading
    from bposit_b200 import ops

    def world(seed):
        cache = make(2, 2, 64, [2100, 60], "bp8", 64, track=True, seed=seed)
        x = [queries(2, n, 64, seed=seed + i) for i, n in enumerate((14, 2, 2))]
        cos = torch.rand(3000, 32, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))

        def step():
            q = ops.kv_append(cache, x[1], x[2], q=x[0], cos=cos, sin=1 - cos)
            out = ops.paged_attention(cache, q, accumulate=True)
            return out, ops.kv_evict(cache, 1500, recent=10, sinks=2)
        return cache, step

    def state(cache):
        return [t.clone() for t in (cache.k, cache.k_exp, cache.v, cache.positions, cache.scores)]

    streams = [torch.cuda.Stream() for _ in range(2)]
    want = []
    for seed in (10, 20):
        cache, step = world(seed)
        want.append([t.clone() for _ in range(3) for t in step()] + state(cache))
    torch.cuda.synchronize()
    for how in ("eager", "threads", "graph"):
        worlds = [world(10), world(20)]
        got = [[], []]
        torch.cuda.synchronize()

        def run(i, times=3):
            with torch.cuda.stream(streams[i]):
                for _ in range(times):
                    got[i] += [t.clone() for t in worlds[i][1]()]
        if how == "eager":
            for i in range(2):
                run(i)
        elif how == "threads":
            threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
            for t in threads:
                t.start()
            for t in threads:
                t.join()
        else:
            graph, main, results = torch.cuda.CUDAGraph(), torch.cuda.Stream(), [None, None]
            with torch.cuda.graph(graph, stream=main):
                for i in range(2):
                    streams[i].wait_stream(main)
                    with torch.cuda.stream(streams[i]):
                        results[i] = worlds[i][1]()
                for s in streams:
                    main.wait_stream(s)
            for _ in range(3):
                graph.replay()
                torch.cuda.synchronize()
                for i in range(2):
                    got[i] += [t.clone() for t in results[i]]
        torch.cuda.synchronize()
        for i in range(2):
            for a, b in zip(got[i] + state(worlds[i][0]), want[i], strict=True):
                assert torch.equal(a, b), (how, i)


def test_cache_tensors_are_written_in_place(orc):
    from bposit_b200 import ops
    from bposit_b200.kv import PagedKVCache
    cache = PagedKVCache(2, 2, 64, 100, track=True)
    with pytest.raises(AttributeError):
        cache.page_table = cache.page_table.clone()
    with pytest.raises(ValueError):
        cache.advance(-1)
    cache.advance(3)
    q = queries(2, 4, 64)
    for layer in (-1, 1, 1 << 32):
        with pytest.raises(ValueError):
            ops.paged_attention(cache, q, layer=layer)
        with pytest.raises(ValueError):
            ops.kv_append(cache, q[:, :2], q[:, 2:], layer=layer)
    for kw in (dict(budget=1 << 32), dict(budget=2, recent=1 << 40), dict(budget=2, sinks=1 << 31)):
        with pytest.raises(ValueError):
            ops.kv_evict(cache, **kw)
    assert torch.equal(ops.paged_attention(cache, q, max_length=(1 << 32) + 1), ops.paged_attention(cache, q))
    for v, kw in ((None, {}), (q[:, 2:], dict(cos=1.0, sin=1.0))):
        with pytest.raises(ValueError):
            ops.kv_append(cache, q[:, :2], v, **kw)


def test_sequences_may_share_pages(orc):
    cache = make(3, 2, 64, [100, 100, 40], "bp8", 16)
    cache.page_table[1, :4] = cache.page_table[0, :4]
    cache.page_table[2, :3] = cache.page_table[0, 0]
    check_attention(orc, cache, queries(3, 4, 64))


def test_attention_reads_views_in_place_and_copies_what_it_must(orc):
    from bposit_b200 import ops
    cache = make(3, 2, 64, [33, 80, 1], "bp8", 16)
    wide = queries(3, 20, 64)
    want = ops.paged_attention(cache, wide[:, :4].contiguous())
    assert torch.equal(ops.paged_attention(cache, wide[:, :4]), want)
    flat = torch.zeros(3 * 4 * 64 + 1, device="cuda")
    odd = flat[1:].view(3, 4, 64)
    odd.copy_(wide[:, :4])
    assert torch.equal(ops.paged_attention(cache, odd), want)
    assert torch.equal(ops.paged_attention(cache, wide[:, :4].transpose(0, 1).contiguous().transpose(0, 1)), want)
    out = torch.empty_like(want)
    assert ops.paged_attention(cache, wide[:, :4], out=out) is out and torch.equal(out, want)


def test_many_sequences_and_one_row_batches(orc):
    lens = [(7 * i) % 90 for i in range(301)]
    cache = make(301, 1, 32, lens, "bp8", 16)
    check_attention(orc, cache, queries(301, 2, 32))


# ---- append ----
@pytest.mark.parametrize("fmt", ["bp8", "bp16"])
@pytest.mark.parametrize("dim,heads,kv_heads,dtype", [(64, 14, 2, torch.float32), (32, 3, 3, torch.float32),
                                                      (96, 8, 1, torch.bfloat16), (128, 5, 5, torch.float16)])
@pytest.mark.parametrize("tokens", [1, 37, 300])
def test_append_is_exact(orc, fmt, dim, heads, kv_heads, dtype, tokens):
    from bposit_b200 import ops
    cache = make(3, kv_heads, dim, [tokens] * 3, fmt, 16, layers=2, track=True)
    g = torch.Generator(device="cuda").manual_seed(tokens)
    x = torch.randn(tokens, (heads + 2 * kv_heads) * dim, generator=g, device="cuda")
    x *= torch.exp2(torch.randint(-12, 12, (tokens, 1), generator=g, device="cuda").float())
    x = x.to(dtype)
    q, k, v = (t.view(tokens, -1, dim) for t in x.split((heads * dim, kv_heads * dim, kv_heads * dim), dim=-1))
    ang = torch.rand(500, dim // 2, generator=g, device="cuda") * 6.3
    cos, sin = ang.cos(), ang.sin()
    pos = torch.randint(0, 500, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    seqs = torch.randint(0, 3, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    places = torch.randperm(tokens, generator=g, device="cuda").to(torch.int32)
    was = [t.clone() for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.positions, cache.scores)]
    got = ops.kv_append(cache, k, v, q=q, cos=cos, sin=sin, positions=pos, seqs=seqs, places=places, layer=1)
    c, s = cos[pos.long()].cpu(), sin[pos.long()].cpu()
    want, tol = ref.rotated_queries(q, c, s)
    assert got.dtype == dtype and (got.double().cpu() - want).abs().le(tol).all()
    page = cache.page_table[seqs.long(), places.long() // 16].long().cpu().numpy()
    off = places.cpu().numpy() % 16
    touched = np.zeros(cache.k.shape[1:4], bool)
    touched[page, :, off] = True
    for pool, exps, x, old in ((cache.k, cache.k_exp, ref.rotate(k, c, s), was[0]),
                               (cache.v, cache.v_exp, v.float().cpu(), was[1])):
        codes, e = ref.encode(orc, x, fmt)
        host = pool.cpu().numpy()
        assert np.array_equal(host[1][page, :, off], codes)
        if e is not None:
            assert np.array_equal(exps[1].cpu().numpy()[page, :, off], e)
        same = (pool.view(torch.uint8) == old).view(2, *touched.shape, -1).all(-1).cpu().numpy()
        assert same[0].all() and same[1][~touched].all()
    b, i = seqs.long(), places.long()
    assert torch.equal(cache.positions[1][b, :, i], pos[:, None].expand(-1, kv_heads))
    assert not cache.scores[1][b, :, i].any()
    cache.positions[1][b, :, i] = was[2][1][b, :, i]
    cache.scores[1][b, :, i] = was[3][1][b, :, i]
    assert torch.equal(cache.positions, was[2]) and torch.equal(cache.scores, was[3])


@pytest.mark.parametrize("fmt", ["bp8", "bp16"])
@pytest.mark.parametrize("dim,heads,kv_heads,dtype", [(64, 14, 2, torch.bfloat16), (32, 20, 1, torch.float16),
                                                      (96, 8, 1, torch.float32), (128, 9, 1, torch.float32)])
def test_append_of_many_tokens(orc, fmt, dim, heads, kv_heads, dtype):
    test_append_is_exact(orc, fmt, dim, heads, kv_heads, dtype, 2999)


@pytest.mark.parametrize("fmt", ["bp8", "bp16"])
def test_append_of_extreme_rows(orc, fmt):
    """Zeros, subnormals, the largest numbers, infinities and NaN, without rotation."""
    from bposit_b200 import ops
    rows = torch.zeros(7, 1, 64)
    rows[1, 0, 3] = 2.0 ** -149
    rows[2, 0, :4] = torch.tensor([3e38, -1e-40, 1.0, -2.0 ** -126])
    rows[3, 0, :3] = torch.tensor([math.inf, -math.inf, 1.5])
    rows[4, 0, :3] = torch.tensor([math.nan, 2.0, -0.0])
    rows[5, 0] = math.inf
    rows[6, 0] = torch.arange(64) * 2.0 ** -140
    cache = make(7, 1, 64, [1, 3, 17, 20, 5, 6, 32], fmt, 16)
    ops.kv_append(cache, rows.cuda(), rows.cuda())
    codes, e = ref.encode(orc, rows, fmt)
    at = cache.lengths.cpu().numpy() - 1
    page = cache.page_table.cpu().numpy()[np.arange(7), at // 16]
    for pool, exps in ((cache.k, cache.k_exp), (cache.v, cache.v_exp)):
        assert np.array_equal(pool.cpu().numpy()[0][page, :, at % 16], codes)
        if e is not None:
            assert np.array_equal(exps.cpu().numpy()[0][page, :, at % 16], e)


def test_append_drops_what_has_no_place(orc):
    from bposit_b200 import ops
    cache = make(2, 2, 64, [0, 30], "bp8", 16, track=True)
    cache.page_table[0, 1] = 1000
    old = [t.clone() for t in (cache.k, cache.v, cache.k_exp, cache.v_exp, cache.positions, cache.scores)]
    k, q = queries(6, 2, 64), queries(6, 4, 64, seed=5)
    ones = torch.ones(4, 32, device="cuda")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    got = ops.kv_append(cache, k, k, q=q, cos=ones, sin=ones * 0, positions=i32(0, 1, 2, 3, 4, -1),
                        seqs=i32(-1, 2, 0, 1, 0, 1 << 30), places=i32(0, 0, -1, cache.capacity, 17, 3))
    assert all(torch.equal(a, b) for a, b in zip(old, (cache.k, cache.v, cache.k_exp, cache.v_exp, cache.positions,
                                                       cache.scores)))
    assert torch.equal(got[:4], q[:4]) and got[4:].isnan().all()      # rows 4 and -1 are not in the tables
    # an empty sequence has no last entry
    ops.kv_append(cache, k[:2], k[:2])
    assert torch.equal(cache.k[0, cache.page_table[0, 0].long()], old[0][0, cache.page_table[0, 0].long()])
    assert cache.positions[0, 1, 0, 29] == 29 and cache.scores[0, 1, 0, 29] == 0


# ---- evict ----
def check_evict(cache, budget, recent, sinks, weights=None, lens=None):
    from bposit_b200 import ops
    lens = cache.lengths.tolist() if lens is None else lens
    w = (cache.scores if weights is None else weights).cpu().numpy()
    pos = cache.positions.cpu().numpy()
    names = ("k", "v", "k_exp", "v_exp")
    old = {n: getattr(cache, n).clone().cpu() for n in names if getattr(cache, n) is not None}
    track = cache.positions.clone().cpu(), cache.scores.clone().cpu()
    keep = ops.kv_evict(cache, budget, recent=recent, sinks=sinks, weights=weights).cpu().numpy()
    table, page = cache.page_table.cpu().numpy(), cache.page_size
    for layer, b, hk in np.ndindex(cache.layers, cache.batch, cache.kv_heads):
        n = lens[b]
        want = ref.evict_keep(pos[layer, b, hk], w[layer, b, hk], n, budget, recent, sinks)
        assert np.array_equal(keep[layer, b, hk], want), (layer, b, hk)
        to = np.nonzero((want != np.arange(budget)) & (want >= 0))[0]
        src = want[to]
        for t in track:
            t[layer, b, hk][to] = t[layer, b, hk][src].clone()
        for pool in old.values():
            p = pool[layer].view(torch.uint8) if pool.dtype != torch.int8 else pool[layer]
            p[table[b, to // page], hk, to % page] = p[table[b, src // page], hk, src % page].clone()
    for n, t in old.items():
        assert torch.equal(getattr(cache, n).cpu().view(torch.uint8), t.view(torch.uint8)), n
    assert torch.equal(cache.positions.cpu(), track[0])
    assert torch.equal(cache.scores.cpu().view(torch.int32), track[1].view(torch.int32))


@pytest.mark.parametrize("fmt,dim", [("bp8", 64), ("bp16", 32), ("bp8", 96), ("bp16", 128)])
@pytest.mark.parametrize("budget,recent,sinks", [(1, 0, 0), (16, 5, 2), (63, 0, 4), (200, 50, 1), (700, 699, 0)])
def test_evict_matches_plain_form(fmt, dim, budget, recent, sinks):
    lens = [0, 1, 17, 64, 201, 1500]
    cache = make(6, 2, dim, lens, fmt, 16, layers=2, track=True, seed=budget)
    check_evict(cache, budget, recent, sinks)


def test_evict_orders_ties_zeros_and_nan():
    cache = make(4, 1, 64, [900, 900, 900, 900], "bp8", 64, track=True)
    w = torch.zeros_like(cache.scores)                    # all equal: the first ones stay
    g = torch.Generator(device="cuda").manual_seed(0)
    w[0, 1] = torch.randint(0, 3, w[0, 1].shape, generator=g, device="cuda")
    w[0, 2] = torch.randn(w[0, 2].shape, generator=g, device="cuda")
    w[0, 2, :, ::7] = math.nan
    w[0, 2, :, 1::7] = -0.0
    w[0, 2, :, 2::7] = 0.0
    w[0, 2, :, 3::21], w[0, 2, :, 10::21] = math.inf, -math.inf
    w[0, 3] = math.nan
    for budget in (1, 255, 512, 600, 800, 899):
        check_evict(cache, budget, 3, 2, weights=w)


def test_evict_with_more_guarded_entries_than_the_budget():
    cache = make(2, 2, 64, [500, 80], "bp8", 16, track=True)
    check_evict(cache, 64, 400, 30)
    cache.positions.fill_(5)                              # every entry is the newest
    check_evict(cache, 40, 1, 0)
    cache.positions.fill_(-(1 << 31))
    check_evict(cache, 30, 0, 0)
    cache.positions.fill_((1 << 31) - 1)
    check_evict(cache, 20, (1 << 31) - 1, (1 << 31) - 1)


@pytest.mark.parametrize("length,budget", [(1024, 1000), (1025, 512), (2048, 3), (2049, 1024), (5000, 4096), (8192, 4096),
                                           (8193, 8192), (16384, 5000), (16385, 8192), (20001, 20000), (33000, 1)])
@pytest.mark.parametrize("kind", ["spread", "ties"])
def test_evict_at_every_capacity(length, budget, kind):
    cache = make(2, 1, 32, [length, budget], "bp8", 16, track=True, seed=length, per=-(-length // 16))
    if kind == "ties":
        g = torch.Generator(device="cuda").manual_seed(budget)
        w = torch.randint(-2, 3, cache.scores.shape, generator=g, device="cuda").float() / 4
        w[..., 5::11], w[..., 6::13], w[..., 7::17] = math.nan, -0.0, math.inf
        cache.scores.copy_(w)
    check_evict(cache, budget, min(40, length // 30), 3)


def test_evict_long_rows_and_own_scores():
    cache = make(1, 1, 32, [40000], "bp8", 128, track=True)
    check_evict(cache, 9000, 100, 4)
    cache.lengths.fill_(9000)
    check_evict(cache, 8999, 100, 4)
    check_evict(cache, 8999, 0, 0, lens=[9000])


def test_evict_with_a_page_outside_the_pool_writes_nothing_there():
    from bposit_b200 import ops
    cache = make(2, 1, 64, [96, 96], "bp8", 16, track=True)
    cache.page_table[0, 5] = -3
    cache.page_table[0, 0] = 999
    w = torch.arange(96, device="cuda", dtype=torch.float32).expand(1, 2, 1, 96).contiguous()
    old = cache.k.clone()
    keep = ops.kv_evict(cache, 32, weights=w)
    assert torch.equal(keep[0, 0], keep[0, 1])
    t = cache.page_table.long().cpu()
    assert torch.equal(cache.k[0, t[1, 0]], old[0, t[1, 4]])   # the other sequence moved
    assert torch.equal(cache.k[0, t[0, 1]], old[0, t[0, 1]])   # sources on the missing page 5
    untouched = sorted(set(range(cache.pages)) - {int(t[1, 0]), int(t[1, 1])})
    assert torch.equal(cache.k[0, untouched], old[0, untouched])


@pytest.mark.parametrize("fmt", ["bp8", "bp16"])
def test_pools_of_more_than_4_gib(fmt):
    """Rows behind 2^32 bytes of codes, in both layers, against a small cache with the same entries."""
    from bposit_b200 import ops
    from bposit_b200.kv import PagedKVCache
    dim, page, heads = 128, 64, 2
    small = make(2, heads, dim, [300, 130], fmt, page, layers=2, track=True)
    pages = (1 << 32) // (heads * page * dim * (1 if fmt == "bp8" else 2)) // 2 + 50   # a layer: 2^31 bytes and more
    shape = (2, pages, heads, page)
    k, v = (torch.empty(shape + (dim,), dtype=small.k.dtype, device="cuda") for _ in range(2))
    ke = ve = None
    if fmt == "bp8":
        ke, ve = (torch.empty(shape, dtype=torch.int8, device="cuda") for _ in range(2))
    move = torch.arange(pages - small.pages, pages, dtype=torch.int32, device="cuda")
    for x, y in ((k, small.k), (v, small.v), (ke, small.k_exp), (ve, small.v_exp)):
        if x is not None:
            x[:, -small.pages:] = y
    big = PagedKVCache.over(k, v, move[small.page_table.long()], small.lengths.clone(), k_exp=ke, v_exp=ve,
                            positions=small.positions.clone(), scores=small.scores.clone())
    new = queries(2, 8, dim, seed=7)
    cos = torch.rand(400, dim // 2, device="cuda")
    results = []
    for c in (small, big):
        out = []
        for layer in (0, 1):
            q = ops.kv_append(c, new[:, :2], new[:, 2:4], q=new[:, 4:], cos=cos, sin=1 - cos, layer=layer)
            out += [q, ops.paged_attention(c, q, layer=layer, accumulate=True)]
        out.append(ops.kv_evict(c, 100, recent=20, sinks=2))
        c.lengths.clamp_(max=100)
        out += [ops.paged_attention(c, q, layer=layer) for layer in (0, 1)] + [c.positions, c.scores]
        results.append(out)
    for a, b in zip(*results, strict=True):
        assert torch.equal(a, b)
    for x, y in ((k, small.k), (v, small.v), (ke, small.k_exp), (ve, small.v_exp)):
        if x is not None:
            assert torch.equal(x[:, -small.pages:].view(torch.uint8), y.view(torch.uint8))
