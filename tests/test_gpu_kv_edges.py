"""Calls at the edges of what the paged key-value cache documents."""
from __future__ import annotations

import math

import pytest
import torch

import kv_reference as ref
from test_gpu_kv import make, queries
from test_gpu_kv_model import small

pytestmark = pytest.mark.gpu


# ---- scores of minus infinity ----
@pytest.mark.parametrize("fmt,dim,page", [("bp8", 64, 64), ("bp16", 128, 16)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("length", [1, 20, 64, 3000])
@pytest.mark.parametrize("sign", [-1, 1])
def test_an_infinite_query_leaves_the_scores(fmt, dim, page, dtype, length, sign):
    """Element 0 of every key is positive, so that one infinite element of a query makes every score of its head
    infinite with one sign: the softmax is NaN whichever it is, in one part or in several."""
    from bposit_b200 import ops
    cache = make(2, 2, dim, [length, 50], fmt, page, track=True)
    (cache.k if fmt == "bp8" else cache.k.view(torch.int16))[..., 0] = 0x50 if fmt == "bp8" else 0x5000
    q = queries(2, 8, dim, dtype)
    good, start = ops.paged_attention(cache, q), cache.scores.clone()
    q[0, 6, 0] = sign * math.inf                    # kv head 1 of sequence 0
    got, lse = ops.paged_attention(cache, q, accumulate=True, return_lse=True)
    assert got[0, 6].isnan().all()
    assert lse[0, 6] == -math.inf if sign < 0 else lse[0, 6].isnan()
    keep = torch.ones(2, 8, dtype=torch.bool, device="cuda")
    keep[0, 6] = False
    assert torch.equal(got[keep], good[keep]) and lse[keep].isfinite().all()
    assert torch.equal(cache.scores[0, 0, 1], start[0, 0, 1]) and cache.scores.isfinite().all()
    assert cache.scores[0, 0, 0, :length].ge(start[0, 0, 0, :length]).all()
    assert cache.scores[0, 0, 0, :length].gt(start[0, 0, 0, :length]).any()


@pytest.mark.parametrize("n", [40, 300, 3000])
def test_scores_that_overflow_downwards_weigh_nothing(orc, n):
    """The first half of the entries has scores near -1e39, which fp32 does not hold; the others count as if they were
    alone, also where whole parts of a long row have no other score."""
    from bposit_b200 import ops
    cache = make(1, 1, 64, [n], "bp8", 64, track=True)
    cache.k_exp.zero_()
    half = n // 2
    for i in range(-(-n // 64)):
        p = int(cache.page_table[0, i])
        lost = (torch.arange(64, device="cuda") + i * 64 < half)
        cache.k[0, p, 0, :, 0] = torch.where(lost, 0x50, 0).to(torch.uint8)
    q = queries(1, 4, 64)
    q[..., 0] = -3e38
    start = cache.scores.clone()
    got, lse = ops.paged_attention(cache, q, accumulate=True, return_lse=True)
    tab = ref.code_values(orc, "bp8")
    k, v = (ref.held(cache, tab, w, 0, 0, 0, n)[half:] for w in ("k", "v"))
    x = q[0].double().cpu()
    s = x @ k.T * 0.125
    p = torch.softmax(s, dim=-1)
    # the terms of kv_reference.attention's bound, of the entries that count (element 0 adds exact zeros to them)
    u = 2.0 ** -24
    ds = 2 * u * (64 + 8) * (x[:, 1:].abs() @ k[:, 1:].abs().T * 0.125).amax(-1) + u * s.abs().amax(-1) * 4
    rel = 2 * ds + u * (400 + n / 32)
    bound = 2 * rel[:, None] * (p @ v.abs())
    want = p @ v
    assert ((got[0].double().cpu() - want).abs() <= bound + u * 1.01 * (want.abs() + bound)).all()
    want = torch.logsumexp(s, dim=-1)
    assert ((lse[0].double().cpu() - want).abs() <= rel + 4 * u * want.abs()).all()
    assert torch.equal(cache.scores[0, 0, 0, :half], start[0, 0, 0, :half])
    want = start[0, 0, 0, half:n].double().cpu() + p.sum(0)
    tol = (2 * rel[:, None] * p).sum(0) + 5 * u * want.abs()
    assert ((cache.scores[0, 0, 0, half:n].double().cpu() - want).abs() <= tol).all()


# ---- lengths behind the capacity ----
def contents(cache):
    return [t.clone().view(torch.uint8) for t in (cache.k, cache.v, cache.k_exp, cache.v_exp, cache.positions,
                                                  cache.scores) if t is not None]


@pytest.mark.parametrize("fmt", ["bp8", "bp16"])
def test_a_token_behind_the_capacity_is_dropped(fmt):
    from bposit_b200 import ops
    cache = make(6, 2, 64, [32] * 6, fmt, 16, track=True)
    cap = cache.capacity
    cache.lengths.copy_(torch.tensor([cap + 1, (1 << 31) - 1, cap, -(1 << 31), cap + 2, -1]))
    old = contents(cache)
    x = queries(6, 8, 64)
    ones = torch.ones(cap + 2, 32, device="cuda")
    got = ops.kv_append(cache, x[:, :2], x[:, 2:4], q=x[:, 4:], cos=ones, sin=ones * 0)
    held = cache.page_table[2].long()               # sequence 2 alone has a last entry
    for was, now in zip(old, contents(cache)):
        if was.shape[1] == cache.pages:
            was[:, held] = now[:, held]
        else:
            was[:, 2] = now[:, 2]
        assert torch.equal(was, now)
    assert cache.positions[0, 2, :, cap - 1].eq(cap - 1).all() and not cache.scores[0, 2, :, cap - 1].any()
    # queries are turned by the token's place: there are rows for cap + 1 and cap + 2, none for the others
    assert torch.equal(got[[0, 2, 4]], x[[0, 2, 4], 4:]) and got[[1, 3, 5]].isnan().all()


def test_steps_replayed_past_the_capacity_lose_no_entry():
    m = small(2)
    g = torch.Generator(device="cuda").manual_seed(8)
    ids = torch.randint(0, 500, (2, 30), generator=g, device="cuda")
    token = torch.randint(0, 500, (2,), generator=g, device="cuda")
    tables = m.rope_tables(64)
    cache = m.new_cache(2, 32, page_size=16, track=True)
    m.prefill(ids, cache, [30, 10])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.step(token, cache, tables)
    for _ in range(2):
        graph.replay()
    full = [t.clone() for t in (cache.k, cache.v, cache.k_exp, cache.v_exp)]
    pages, pos = cache.page_table[0].long(), cache.positions[:, 0].clone()
    for _ in range(3):
        graph.replay()
    assert cache.lengths.tolist() == [35, 15]
    for was, now in zip(full, (cache.k, cache.v, cache.k_exp, cache.v_exp)):
        assert torch.equal(was[:, pages], now[:, pages])
    assert torch.equal(pos, cache.positions[:, 0])
    assert cache.positions[:, 1, :, :15].eq(torch.arange(15, device="cuda")).all()


# ---- lengths that the host does not know ----
def test_sequences_that_grow_in_turn_fill_the_cache():
    from bposit_b200.kv import PagedKVCache
    cache = PagedKVCache(2, 1, 64, 64, page_size=16)
    for n in ([30, 0], [0, 40], [34, 0], [0, 24]):
        cache.advance(torch.tensor(n, dtype=torch.int32, device="cuda"), most=max(n))
    assert cache.lengths.tolist() == [64, 64] and cache.seen.tolist() == [64, 64] and cache.longest == 64
    for n, most in ((1, None), (torch.tensor([0, 1], dtype=torch.int32, device="cuda"), 1)):
        with pytest.raises(ValueError, match="capacity"):
            cache.advance(n, most=most)
    assert cache.lengths.tolist() == [64, 64] and cache.longest == 64
    cache.lengths[0], cache.seen[0] = 0, 0              # one sequence ends, another starts in its place
    cache.advance(torch.tensor([20, 0], dtype=torch.int32, device="cuda"), most=20)
    assert cache.lengths.tolist() == [20, 64] and cache.longest == 64
    for n, most in ((1 << 40, None), (torch.tensor([45, 0], dtype=torch.int32, device="cuda"), 1 << 40),
                    (torch.full((2,), (1 << 31) - 1, dtype=torch.int32, device="cuda"), (1 << 31) - 1)):
        with pytest.raises(ValueError, match="capacity"):
            cache.advance(n, most=most)
    cache.advance(torch.tensor([44, 0], dtype=torch.int32, device="cuda"), most=1 << 40)
    assert cache.lengths.tolist() == [64, 64]


def test_a_cache_over_tensors_finds_its_room():
    cache = make(2, 2, 64, [30, 5], "bp8", 16)          # capacity 32
    cache.advance(2)
    assert cache.lengths.tolist() == [32, 7] and cache.longest == 32
    with pytest.raises(ValueError, match="capacity"):
        cache.advance()
    assert not cache.is_empty()
    cache.lengths.zero_()
    assert cache.is_empty()


def test_the_host_looks_at_the_lengths_once_they_were_captured():
    m = small(1)
    g = torch.Generator(device="cuda").manual_seed(9)
    ids = torch.randint(0, 500, (2, 20), generator=g, device="cuda")
    token = torch.randint(0, 500, (2,), generator=g, device="cuda")
    tables = m.rope_tables(64)
    cache = m.new_cache(2, 32, page_size=16, track=True)
    m.prefill(ids, cache, [20, 10])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.step(token, cache, tables)
    for _ in range(11):
        graph.replay()
    m.step(token, cache, tables)
    assert cache.lengths.tolist() == [32, 22] and cache.longest == 32
    with pytest.raises(ValueError, match="capacity"):
        m.step(token, cache, tables)
    assert cache.lengths.tolist() == [32, 22]
    cache.evict(29, recent=4, sinks=1)
    assert cache.lengths.tolist() == [29, 22] and cache.longest == 29
    cache.reset()
    graph.replay()
    cache.evict(16)
    assert cache.longest >= 1                           # still a bound
    with pytest.raises(ValueError, match="empty"):
        m.prefill(ids, cache)
    cache.reset()
    m.prefill(ids, cache)
    assert cache.lengths.tolist() == [20, 20] and cache.longest == 20


def test_captures_do_not_use_up_the_room():
    """A captured call moves no length until it is replayed: more of them than entries fit are still captured."""
    from bposit_b200.kv import PagedKVCache
    cache = PagedKVCache(1, 1, 64, 16, page_size=16)
    cache.advance(14)
    graphs = [torch.cuda.CUDAGraph() for _ in range(4)]
    for graph in graphs:
        with torch.cuda.graph(graph):
            cache.advance()
    assert cache.lengths.tolist() == [14] and cache.longest == 16
    cache.advance()
    assert cache.lengths.tolist() == [15] and cache.longest == 15
    graphs[3].replay()
    assert cache.lengths.tolist() == [16]
    with pytest.raises(ValueError, match="capacity"):
        cache.advance()


def test_an_empty_cache_has_a_bound():
    from bposit_b200 import ops
    from bposit_b200.kv import PagedKVCache
    cache = PagedKVCache(2, 2, 64, 64)
    out = ops.paged_attention(cache, queries(2, 4, 64), max_length=cache.bound)
    assert not out.any()


# ---- small budgets ----
@pytest.mark.parametrize("budget", [1, 2, 5, 12, 30, 67])
def test_a_small_budget_keeps_the_newest_tokens(budget, monkeypatch):
    from bposit_b200.kv import PagedKVCache
    cuts = []
    evict = PagedKVCache.evict

    def watched(self, *a, **kw):
        keep = evict(self, *a, **kw)
        first = self.seen - self.lengths.clamp(max=1)       # position of each row's newest token
        cuts.append((self.positions[..., :budget] == first[None, :, None, None]).any(-1).all().item())
        return keep

    monkeypatch.setattr(PagedKVCache, "evict", watched)
    m = small(2)
    g = torch.Generator(device="cuda").manual_seed(10)
    ids = torch.randint(0, 500, (2, 70), generator=g, device="cuda")
    assert m.generate(ids, 40, lengths=[70, 50], page_size=16, budget=budget).shape == (2, 40)
    assert len(cuts) >= 2 and all(cuts)


def test_a_budget_below_what_it_must_keep_is_refused():
    m = small(1)
    ids = torch.zeros(1, 8, dtype=torch.int64, device="cuda")
    for kw in (dict(recent=21, sinks=4), dict(recent=24, sinks=1), dict(sinks=25), dict(recent=25),
               dict(recent=-1), dict(sinks=-1), dict(recent=1 << 40)):
        with pytest.raises(ValueError):
            m.generate(ids, 4, budget=24, **kw)
    assert m.generate(ids, 2, budget=24, recent=20, sinks=4).shape == (1, 2)
    assert m.generate(ids, 2, budget=24, recent=24, sinks=0).shape == (1, 2)


# ---- calls that a model refuses before it moves a length ----
def test_steps_that_cannot_be_taken_leave_the_cache_alone():
    from bposit_b200.kv import PagedKVCache
    m = small(2)
    ids = torch.zeros(2, 8, dtype=torch.int64, device="cuda")
    token, tables = ids[:, 0], m.rope_tables(64)
    cache = m.new_cache(2, 32, page_size=16)
    m.prefill(ids, cache)
    for bad in (ids[:1, 0], torch.zeros(3, dtype=torch.int64, device="cuda"), ids):
        with pytest.raises(ValueError, match="ids"):
            m.step(bad, cache, tables)
    assert cache.lengths.tolist() == [8, 8] and cache.seen.tolist() == [8, 8] and cache.longest == 8
    over = make(2, 2, 64, [8, 3], "bp8", 16, layers=2)  # over tensors: it has no count of the tokens seen
    with pytest.raises(ValueError, match="seen"):
        m.step(token, over, tables)
    assert over.lengths.tolist() == [8, 3]
    for other in (PagedKVCache(2, 1, 64, 32, layers=2), PagedKVCache(2, 2, 32, 32, layers=2), PagedKVCache(2, 2, 64, 32)):
        for call in (lambda: m.step(token, other, tables), lambda: m.prefill(ids, other)):
            with pytest.raises(ValueError, match="cache"):
                call()
        assert not other.lengths.any() and other.longest == 0


# ---- the value of every code ----
def blocks(fmt, dim, n):
    """Pools of one layer whose row (sequence b, kv head h, entry i) holds `dim` codes that follow one another, turned
    by i, so that all rows together hold every code at every entry: (codes [batch, 8, n, dim], cache)."""
    from bposit_b200.kv import PagedKVCache
    codes, heads = (256, 2) if fmt == "bp8" else (65536, 8)
    batch = codes // (heads * dim)
    first = (torch.arange(batch * heads, device="cuda") * dim).view(batch, heads, 1, 1)
    turn = torch.arange(n, device="cuda")[:, None] + torch.arange(dim, device="cuda")
    c = first + turn % dim
    dt = torch.uint8 if fmt == "bp8" else torch.int16
    pool = torch.zeros(batch, heads, 64, dim, dtype=dt, device="cuda")
    pool[:, :, :n] = (c if fmt == "bp8" else (c + 32768) % 65536 - 32768).to(dt)
    pool = pool[None] if fmt == "bp8" else pool[None].view(torch.uint16)
    exps = {}
    if fmt == "bp8":
        exps = {k: torch.zeros(1, batch, heads, 64, dtype=torch.int8, device="cuda") for k in ("k_exp", "v_exp")}
    table = torch.arange(batch, dtype=torch.int32, device="cuda")[:, None].contiguous()
    lengths = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    other = torch.zeros_like(pool.view(dt)).view(pool.dtype)
    return c, pool, other, lambda k, v: PagedKVCache.over(k, v, table, lengths, **exps)


CODES = [("bp8", 32), ("bp8", 64), ("bp8", 128), ("bp16", 32), ("bp16", 64), ("bp16", 96), ("bp16", 128)]


@pytest.mark.parametrize("fmt,dim", [c for c in CODES if c[1] != 96])
@pytest.mark.parametrize("n", [1, 64])
def test_the_value_of_every_code(orc, fmt, dim, n):
    """One entry has the weight 1 and the others 0, both exactly, so the output is the values of its codes: one entry
    in a unit by itself, or one of a whole tile of codes of its block."""
    from bposit_b200 import ops
    c, values, keys, over = blocks(fmt, dim, n)
    batch, heads = c.shape[:2]
    # key element 0 is 1.0 in the chosen entry and 0 in the others: 300 apart in the exponent of 2, e^-300 is 0 in fp32
    chosen = (torch.arange(batch * heads, device="cuda") * 7 % n).view(batch, heads)
    plain = keys if fmt == "bp8" else keys.view(torch.int16)
    plain[0, torch.arange(batch, device="cuda")[:, None], torch.arange(heads, device="cuda"), chosen, 0] = \
        0x40 if fmt == "bp8" else 0x4000
    q = torch.zeros(batch, heads, dim, device="cuda")
    q[..., 0] = 300.0
    out = ops.paged_attention(over(keys, values), q, scale=1.0)
    tab = ref.code_values(orc, fmt).float().cuda()
    want = tab[torch.gather(c, 2, chosen[:, :, None, None].expand(-1, -1, 1, dim))[:, :, 0]]
    assert torch.equal(out, want)


@pytest.mark.parametrize("fmt,dim", [c for c in CODES if c[1] != 96])
@pytest.mark.parametrize("n", [1, 64])
def test_the_score_of_every_code(orc, fmt, dim, n):
    """A query head for each column of the keys, with 1 over the power of two of the code there and 0 elsewhere: the
    score is the code's value between 1 and 2, and the logarithm of the denominator shows it, with one entry or with
    a tile of equal ones."""
    from bposit_b200 import ops
    c, keys, values, over = blocks(fmt, dim, n)
    batch, heads = c.shape[:2]
    if n > 1:
        # every entry of a row holds the same codes
        plain = keys if fmt == "bp8" else keys.view(torch.int16)
        plain.copy_(plain[:, :, :, :1].expand(plain.shape).clone())
    tab = ref.code_values(orc, fmt)
    v = tab[c[:, :, 0].cpu()]                                    # [batch, heads, dim]
    size = torch.where(v == 0, 0.0, torch.exp2(1.0 - torch.frexp(v)[1].double()))
    q = torch.zeros(batch, heads * dim, dim, dtype=torch.float64)
    at = torch.arange(dim).repeat(heads)
    q[:, torch.arange(heads * dim), at] = size.reshape(batch, -1)
    _, lse = ops.paged_attention(over(keys, values), q.float().cuda(), scale=1.0, return_lse=True)
    score = (v * size).reshape(batch, -1)                        # 0, or from 1 to 2 in magnitude
    want = score + math.log(n)
    # half steps: of log2(e) and ln 2 as fp32 numbers, the products with them, the sum with log2(n), at most 9 in base
    # 2: codes are told apart by 2^-11
    tol = 2.0 ** -24 * (4 * want.abs() + 9)
    assert ((lse.double().cpu() - want).abs() <= tol).all()
