"""Workloads of the paged b-posit key-value cache: writing rotated tokens into it, attending
to it with one new token per sequence, and evicting entries by accumulated attention weight.

The cache holds keys and values as bp8 codes with one power-of-two exponent per (token, kv
head), or as bp16 codes, in pages of `page` tokens: pools [layers, pages, kv_heads, page, dim],
a page table [batch, max_pages], and per (layer, sequence, kv head) the entries' positions and
accumulated attention weights.  With `own` false, run() computes each operator from elementary
torch operations; with `own` true it calls the library.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

_DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------ cases ---
def listed():
    A = dict(op="attend", track=False, page=64)
    return [
        # one chat in its first words, the latency of a decode step: Qwen2.5-0.5B-shaped heads
        dict(A, name="attend_first_words", batch=1, length=17, heads=14, kv_heads=2, dim=64, fmt="bp8", dtype="fp32"),
        # a few chats of ordinary lengths
        dict(A, name="attend_chats", batch=8, length=1500, heads=14, kv_heads=2, dim=64, fmt="bp8", dtype="fp32"),
        # one sequence with a whole book before it: split over the cache's length
        dict(A, name="attend_one_long", batch=1, length=131071, heads=14, kv_heads=2, dim=64, fmt="bp8", dtype="fp32"),
        # a serving batch, short and long sequences mixed
        dict(A, name="attend_serving", batch=64, length=16384, heads=14, kv_heads=2, dim=64, fmt="bp8", dtype="fp32"),
        # wide heads of a larger model in the 16-bit format, bf16 activations, small pages
        dict(A, name="attend_bp16_wide", batch=16, length=4096, heads=32, kv_heads=8, dim=128, fmt="bp16",
             dtype="bf16", page=16),
        # SmolLM2-135M-shaped heads, keeping the weight that each entry has received
        dict(A, name="attend_weights", batch=16, length=4096, heads=9, kv_heads=3, dim=64, fmt="bp8", dtype="fp32",
             track=True),
        # the decode step's write: one token per sequence
        dict(op="append", name="append_step", tokens=16, batch=16, heads=14, kv_heads=2, dim=64, fmt="bp8",
             dtype="fp32", page=64),
        # a prompt batch of 8 x 1024 tokens, the shape of the model forward
        dict(op="append", name="append_prompts", tokens=8192, batch=8, heads=14, kv_heads=2, dim=64, fmt="bp8",
             dtype="fp32", page=64),
        # a large prompt batch with bf16 activations in the 16-bit format, an odd number of tokens
        dict(op="append", name="append_bp16", tokens=20001, batch=5, heads=9, kv_heads=3, dim=64, fmt="bp16",
             dtype="bf16", page=32),
        # a bounded cache during generation: a page of new entries pushes the least used out
        dict(op="evict", name="evict_step", layers=24, batch=8, length=1088, budget=1024, recent=64, sinks=4,
             kv_heads=2, dim=64, fmt="bp8", page=64),
        # a long prompt cut down to its most attended entries
        dict(op="evict", name="evict_prompt", layers=24, batch=4, length=8192, budget=2048, recent=256, sinks=4,
             kv_heads=2, dim=64, fmt="bp8", page=64),
        # one sequence, one layer, a single entry over the budget
        dict(op="evict", name="evict_one", layers=1, batch=1, length=513, budget=512, recent=32, sinks=1,
             kv_heads=2, dim=64, fmt="bp16", page=16),
    ]


_HEADS = ((14, 2), (9, 3), (32, 8), (8, 8), (12, 4), (16, 1), (5, 5))


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("attend", "attend", "append", "evict"))
    heads, kv_heads = rng.choice(_HEADS)
    fmt = rng.choice(("bp8", "bp8", "bp16"))
    dim = rng.choice((32, 64, 64, 96, 128))
    page = rng.choice((16, 32, 64, 128))
    nb = 1 if fmt == "bp8" else 2
    if op == "attend":
        length = _log(rng, 1, 65536)
        batch = max(1, min(_log(rng, 1, 64), (1 << 28) // (length * kv_heads * dim * nb * 2)))
        return dict(op=op, batch=batch, length=length, heads=heads, kv_heads=kv_heads, dim=dim, fmt=fmt,
                    dtype=rng.choice(("fp32", "fp32", "bf16", "fp16")), page=page, track=rng.random() < 0.4)
    if op == "append":
        tokens = _log(rng, 1, 12000)
        return dict(op=op, tokens=tokens, batch=min(tokens, _log(rng, 1, 32)), heads=heads, kv_heads=kv_heads,
                    dim=dim, fmt=fmt, dtype=rng.choice(("fp32", "bf16", "fp16")), page=page)
    length = _log(rng, 2, 8192)
    kv_heads = min(kv_heads, 3)
    layers = rng.choice((1, 2, 12, 24))
    batch = max(1, min(_log(rng, 1, 16), (1 << 26) // (layers * length * kv_heads * dim * nb)))
    budget = max(1, min(length, int(length * rng.uniform(0.1, 1.0))))
    return dict(op=op, layers=layers, batch=batch, length=length, budget=budget, recent=_log(rng, 1, length),
                sinks=rng.choice((0, 1, 4)), kv_heads=kv_heads, dim=dim, fmt=fmt, page=page)


# ------------------------------------------------------- the two formats ---
def _magnitudes(nbits, es, device):
    """float64 values of the positive codes 0 .. 2^(nbits-1) - 1: regime run, es exponent bits
    (left-aligned where the regime leaves fewer), fraction."""
    f = torch.arange(1 << (nbits - 1), dtype=torch.int64, device=device)
    width = nbits - 1
    lead = (f >> (width - 1)) & 1
    rest = torch.where(lead == 1, ~f & ((1 << width) - 1), f)
    run = width - torch.frexp(rest.double()).exponent.long()      # leading bits equal to `lead`
    k = torch.where(lead == 1, run - 1, -run)
    rem = (width - 1 - run).clamp(min=0)
    tail = f & ((1 << rem) - 1)
    ew = rem.clamp(max=es)
    fw = rem - ew
    e = (tail >> fw) << (es - ew)
    frac = (tail & ((1 << fw) - 1)).double() / (1 << fw).double()
    v = torch.ldexp(1.0 + frac, k * (1 << es) + e)
    v[0] = 0.0
    return v


_TABLES: dict = {}


def _table(fmt, device):
    """fp32 value of every code (zero and NaR count as zero)."""
    key = (fmt, str(device))
    if key not in _TABLES:
        mag = _magnitudes(8, 2, device) if fmt == "bp8" else _magnitudes(16, 3, device)
        n = mag.numel()
        _TABLES[key] = torch.cat((mag, torch.zeros(1, dtype=mag.dtype, device=device), -mag[1:].flip(0))).float()
        assert _TABLES[key].numel() == 2 * n
    return _TABLES[key]


def _bits(codes):
    return codes.to(torch.int64) & (0xFF if codes.dtype == torch.uint8 else 0xFFFF)


def _encode_bp8(x):
    """int64 codes of float64 values: nearest, ties to the smaller magnitude, nonzero stays nonzero."""
    mag = _magnitudes(8, 2, x.device)
    mids = (mag[1:-1] + mag[2:]) / 2
    m = torch.bucketize(x.abs(), mids) + (x != 0)
    return torch.where(x < 0, 256 - m, m) & 0xFF


def _encode_bp16(x):
    """int64 codes of fp32 values: the bit string of regime, exponent and fraction, rounded to nearest even."""
    u = x.view(torch.int32).to(torch.int64)
    a = u & 0x7FFFFFFF
    E, M = (a >> 23) - 127, a & 0x7FFFFF
    k, e = E >> 3, E & 7
    run = torch.where(k >= 0, k + 2, 1 - k)
    avail = (15 - run).clamp(min=1)
    eb = avail.clamp(max=3)
    fb = avail - eb
    regime = torch.where(k >= 0, ((1 << (k.clamp(min=0) + 1)) - 1) << 1, torch.ones_like(k))
    field = (regime << avail) | ((e >> (3 - eb)) << fb) | (M >> (23 - fb))
    up = ((M >> (22 - fb)) & 1) & (((M & ((1 << (22 - fb)) - 1)) != 0) | (field & 1 == 1))
    field = (field + up).clamp(max=0x7FFF)
    field = torch.where(run >= 15, torch.where(k >= 14, 0x7FFF, torch.where(k >= 0, 0x7FFE, 1)), field)
    field = torch.where(E > 112, 0x7FFF, torch.where(E < -112, 1, field))
    field = torch.where(a == 0, 0, field)
    return torch.where(u < 0, -field, field) & 0xFFFF


def _encode(x, fmt):
    """fp32 rows [..., dim] -> (codes, exponent of each row): bp8 rows are scaled by a power of two that
    takes the largest magnitude into [8, 16), where the format holds the rows' upper 2^8 with 3 bits of
    fraction; bp16 rows are not scaled."""
    if fmt == "bp16":
        return _encode_bp16(x.contiguous()).to(torch.int16), None
    top = x.abs().amax(-1).double()
    e = torch.where(top > 0, (torch.frexp(top).exponent - 4).clamp(min=-126), 0)
    return _encode_bp8(torch.ldexp(x.double(), -e[..., None])).to(torch.uint8), e.to(torch.int8)


# ---------------------------------------------------------------- inputs ---
def _lengths(c, g):
    """Sequence lengths of a batch: uniform in [1, length], one of the full length, and in batches of
    four and more one that is empty."""
    n = torch.randint(1, c["length"] + 1, (c["batch"],), generator=g, device="cuda")
    n[0] = c["length"]
    if c["batch"] >= 4:
        n[-1] = 0
    return n.to(torch.int32)


def _pool(c, layers, pages, g, fill):
    """Code pools of a cache (and exponents): rows as a model's keys and values come, of normal values."""
    shape = (layers, pages, c["kv_heads"], c["page"], c["dim"])
    dt = torch.uint8 if c["fmt"] == "bp8" else torch.int16
    if not fill:
        k, v = (torch.zeros(shape, dtype=dt, device="cuda") for _ in range(2))
    else:
        x = torch.randn(1 << 18, generator=g, device="cuda") * (4.0 if c["fmt"] == "bp8" else 1.0)
        x = (_encode_bp8(x.double()) if c["fmt"] == "bp8" else _encode_bp16(x)).to(dt)
        k, v = (x[torch.randint(0, x.numel(), (math.prod(shape),), generator=g, device="cuda", dtype=torch.int32)]
                .view(shape) for _ in range(2))
    ke = ve = None
    if c["fmt"] == "bp8":
        ke, ve = (torch.randint(-3, 0, shape[:-1], generator=g, device="cuda", dtype=torch.int8) if fill else
                  torch.zeros(shape[:-1], dtype=torch.int8, device="cuda") for _ in range(2))
    return k, v, ke, ve


def _page_table(batch, per, g):
    """Pages of the pool in no order, a few of them unused."""
    total = batch * per + 3
    return torch.randperm(total, generator=g, device="cuda")[: batch * per].view(batch, per).to(torch.int32), total


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"c": c}
    page = c["page"]
    if c["op"] == "attend":
        per, layers = -(-c["length"] // page), 1
        lengths = _lengths(c, g)
    elif c["op"] == "append":
        layers = 1
        # sequences of uneven lengths: the borders of an even split, each moved by up to 0.4 of a sequence
        mean = c["tokens"] / c["batch"]
        borders = torch.arange(1, c["batch"], device="cuda") + (torch.rand(c["batch"] - 1, generator=g, device="cuda") - 0.5) * 0.8
        edge = torch.tensor([0], device="cuda")
        starts = torch.cat((edge, (borders * mean).long()))
        n = torch.diff(torch.cat((starts, edge + c["tokens"])))
        per = -(-int(1.8 * mean + 2) // page) if c["tokens"] > c["batch"] else 4
        if c["tokens"] == c["batch"]:      # a step: one token behind each sequence's own past
            past = torch.randint(0, per * page, (c["batch"],), generator=g, device="cuda")
            s["seqs"] = s["places"] = None
            positions, lengths = past, past + 1
        else:
            seqs = torch.repeat_interleave(torch.arange(c["batch"], device="cuda"), n)
            positions = torch.arange(c["tokens"], device="cuda") - starts[seqs]
            s["seqs"], s["places"], lengths = seqs.to(torch.int32), positions.to(torch.int32), n
        s["positions"], lengths = positions.to(torch.int32), lengths.to(torch.int32)
    else:
        layers, per = c["layers"], -(-c["length"] // page)
        lengths = torch.full((c["batch"],), c["length"], dtype=torch.int32, device="cuda")
    table, pages = _page_table(c["batch"], per, g)
    k, v, ke, ve = _pool(c, layers, pages, g, c["op"] != "append")
    cap = per * page
    shape = (layers, c["batch"], c["kv_heads"], cap)
    tracked = c["op"] == "evict" or c.get("track", False)
    s.update(k=k, v=v, k_exp=ke, v_exp=ve, page_table=table, lengths=lengths, track=None, scores=None)
    if tracked:
        s["scores"] = torch.rand(shape, generator=g, device="cuda")
        s["track"] = torch.arange(cap, device="cuda", dtype=torch.int32).expand(shape).contiguous()
    dt = _DT[c.get("dtype", "fp32")]
    if c["op"] == "attend":
        s["q"] = torch.randn(c["batch"], c["heads"], c["dim"], generator=g, device="cuda").to(dt)
    elif c["op"] == "append":
        H, N, D = c["heads"], c["kv_heads"], c["dim"]
        # the fused projection's output: q, k and v are views of it
        qkv = torch.randn(c["tokens"], (H + 2 * N) * D, generator=g, device="cuda").to(dt)
        q, kk, vv = qkv.split((H * D, N * D, N * D), dim=-1)
        s["q"], s["new_k"], s["new_v"] = q.view(-1, H, D), kk.view(-1, N, D), vv.view(-1, N, D)
        inv = 1.0 / 1e6 ** (torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
        ang = torch.outer(torch.arange(max(cap, c["tokens"]), device="cuda", dtype=torch.float64), inv)
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    else:
        # what the last tokens of the prompt gave to each entry: a few are attended to far more than most
        s["weights"] = torch.rand(shape, generator=g, device="cuda").pow(8)
    if own:
        from_repo = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "open-bposit_b200")
        if from_repo not in sys.path:
            sys.path.insert(0, from_repo)
        from bposit_b200 import kv
        dt16 = (lambda t: t.view(torch.uint16)) if c["fmt"] == "bp16" else (lambda t: t)
        s["cache"] = kv.PagedKVCache.over(dt16(k), dt16(v), table, lengths, k_exp=ke, v_exp=ve,
                                          positions=s["track"], scores=s["scores"])
    return s


# ----------------------------------------------------------- plain forms ---
def _flat(s, rows_b, places):
    """Index into the pools' [pages * page] view of a sequence's entries."""
    page = s["c"]["page"]
    return s["page_table"].long()[rows_b, places // page] * page + places % page


def _values(s, codes, exps):
    x = _table(s["c"]["fmt"], codes.device)[_bits(codes)]
    return x if exps is None else torch.ldexp(x, exps.int()[..., None])


def _attend(s):
    c = s["c"]
    B, N, D, page = c["batch"], c["kv_heads"], c["dim"], c["page"]
    pt = s["page_table"].long()
    L = pt.shape[1] * page

    def held(codes, exps):       # [B, N, L, D] fp32
        x = codes[0][pt].transpose(1, 2).reshape(B, N, L, D)
        e = None if exps is None else exps[0][pt].transpose(1, 2).reshape(B, N, L)
        return _values(s, x, e)

    q = s["q"].float().view(B, N, c["heads"] // N, D)
    t = torch.matmul(q, held(s["k"], s["k_exp"]).transpose(2, 3)) * (1.0 / math.sqrt(D))
    there = (torch.arange(L, device=q.device) < s["lengths"][:, None])[:, None, None]
    t = torch.where(there, t, -math.inf)
    m = t.amax(-1, keepdim=True)
    p = torch.exp(t - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = torch.matmul(p, held(s["v"], s["v_exp"])).reshape(B, c["heads"], D).to(s["q"].dtype)
    if not c["track"]:
        return {"out": o}
    s["scores"][0] += p.sum(2)
    return {"out": o, "scores": s["scores"]}


def _rotate(x, cos, sin):
    """Rotary positions on the pairs (i, i + dim/2), in float64 from the fp32 tables, rounded to fp32."""
    x = x.double()
    a, b = x.chunk(2, dim=-1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1).float()


def _append(s):
    c = s["c"]
    cos, sin = (t[s["positions"].long()].double()[:, None] for t in (s["cos"], s["sin"]))
    q = _rotate(s["q"], cos, sin).to(s["q"].dtype)
    if s["seqs"] is None:
        at = _flat(s, torch.arange(c["batch"], device=q.device), s["lengths"].long() - 1)
    else:
        at = _flat(s, s["seqs"].long(), s["places"].long())
    page, off = at // c["page"], at % c["page"]
    for pool, exps, x in ((s["k"], s["k_exp"], _rotate(s["new_k"], cos, sin)), (s["v"], s["v_exp"], s["new_v"].float())):
        codes, e = _encode(x, c["fmt"])
        pool[0][page, :, off] = codes
        if e is not None:
            exps[0][page, :, off] = e
    return {"q": q, "k": s["k"], "v": s["v"], "k_exp": s["k_exp"], "v_exp": s["v_exp"]}


def _evict(s):
    c = s["c"]
    Ly, B, N, L, M = c["layers"], c["batch"], c["kv_heads"], c["length"], c["budget"]
    pos, w = s["track"][..., :L], s["weights"][..., :L]
    kept_for_place = (pos < c["sinks"]) | (pos > pos.amax(-1, keepdim=True) - c["recent"])
    key = torch.where(kept_for_place, math.inf, w)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :M]
    kept = torch.zeros(key.shape, dtype=torch.bool, device=key.device).scatter_(-1, order, True)
    # kept entries behind the budget move, in order, into the places in front that were given up
    place = torch.arange(L, device=key.device).expand(key.shape)
    hole, mover = ~kept & (place < M), kept & (place >= M)
    keep = place[..., :M].clone()
    keep[hole[..., :M]] = place[mover]      # both in row order, as many holes as movers in each row
    rows = torch.arange(B, device=key.device)[None, :, None, None].expand(Ly, B, N, M)
    at_l = torch.arange(Ly, device=key.device)[:, None, None, None]
    at_n = torch.arange(N, device=key.device)[None, None, :, None]
    src, dst = _flat(s, rows, keep), _flat(s, rows, place[..., :M])
    page = c["page"]
    for pool in (s["k"], s["v"], s["k_exp"], s["v_exp"]):
        if pool is not None:
            pool[at_l, dst // page, at_n, dst % page] = pool[at_l, src // page, at_n, src % page]
    for t in (s["scores"], s["track"]):
        t[..., :M] = torch.gather(t, -1, keep)
    return {"keep": keep.to(torch.int32), "k": s["k"], "v": s["v"], "k_exp": s["k_exp"], "v_exp": s["v_exp"],
            "scores": s["scores"], "positions": s["track"]}


def run(state):
    s, c = state, state["c"]
    if not own:
        return {"attend": _attend, "append": _append, "evict": _evict}[c["op"]](s)
    from bposit_b200 import ops
    if c["op"] == "attend":
        o = ops.paged_attention(s["cache"], s["q"], accumulate=c["track"])
        return {"out": o, "scores": s["scores"]} if c["track"] else {"out": o}
    if c["op"] == "append":
        q = ops.kv_append(s["cache"], s["new_k"], s["new_v"], q=s["q"], cos=s["cos"], sin=s["sin"],
                          positions=s["positions"], seqs=s["seqs"], places=s["places"])
        return {"q": q, "k": s["k"], "v": s["v"], "k_exp": s["k_exp"], "v_exp": s["v_exp"]}
    keep = ops.kv_evict(s["cache"], c["budget"], recent=c["recent"], sinks=c["sinks"], weights=s["weights"])
    return {"keep": keep, "k": s["k"], "v": s["v"], "k_exp": s["k_exp"], "v_exp": s["v_exp"],
            "scores": s["scores"], "positions": s["track"]}


# ------------------------------------------------------------------ work ---
def work(case):
    c = case
    nb = 1 if c["fmt"] == "bp8" else 2
    row = c["dim"] * nb + (1 if c["fmt"] == "bp8" else 0)      # one token's key or value of one head
    ab = 4 if c.get("dtype", "fp32") == "fp32" else 2
    if c["op"] == "attend":
        # expected entries of the lengths that _lengths draws
        n = c["length"] + (c["batch"] - 1 - (c["batch"] >= 4)) * (c["length"] + 1) / 2
        byt = n * c["kv_heads"] * (2 * row + (8 if c["track"] else 0)) + 2 * c["batch"] * c["heads"] * c["dim"] * ab
        byt += 4 * n / c["page"]
        return {"bytes": byt, "flops": 4.0 * n * c["heads"] * c["dim"]}
    if c["op"] == "append":
        t = c["tokens"]
        vals = t * c["dim"] * (c["heads"] + 2 * c["kv_heads"])
        byt = vals * ab + t * c["heads"] * c["dim"] * ab + 2 * t * c["kv_heads"] * row + 12 * t + 4 * t * c["dim"]
        return {"bytes": byt, "flops": 3.0 * t * c["dim"] * (c["heads"] + c["kv_heads"])}
    rows = c["layers"] * c["batch"] * c["kv_heads"]
    # entries that are kept from behind the budget, if the weights say nothing about the place
    behind = c["length"] - c["budget"]
    fixed = min(behind, c["recent"])
    free = max(0, min(c["budget"], c["length"] - fixed) - fixed)
    moved = fixed + (behind - fixed) * free / max(1, c["length"] - fixed)
    byt = rows * (8 * c["length"] + 4 * c["budget"] + 2 * moved * (2 * row + 8))
    return {"bytes": byt, "flops": 1.0 * rows * c["length"]}


# ----------------------------------------------------------------- exact ---
def _exact_table(fmt):
    """float64 value of every code, bit by bit."""
    nb, es = (8, 2) if fmt == "bp8" else (16, 3)
    out = np.zeros(1 << nb)
    for code in range(1, 1 << nb):
        if code == 1 << (nb - 1):
            continue
        neg = code >> (nb - 1)
        bits = format((1 << nb) - code if neg else code, "0%db" % nb)[1:]
        first = bits[0]
        run = len(bits) - len(bits.lstrip(first))
        k = run - 1 if first == "1" else -run
        tail = bits[run + 1:]
        e = int(tail[:es].ljust(es, "0") or "0", 2)
        f = tail[es:]
        val = (1.0 + (int(f, 2) / (1 << len(f)) if f else 0.0)) * 2.0 ** (k * (1 << es) + e)
        out[code] = -val if neg else val
    return torch.from_numpy(out).cuda()


def exact(case, seed):
    """Attention from its definition, one sequence at a time; the rotated queries; the moved weights; codes,
    exponents and places have none: they are whole values."""
    c = case
    s = prepare(c, seed)
    if c["op"] == "attend":
        tab = _exact_table(c["fmt"])
        B, H, N, D, page = c["batch"], c["heads"], c["kv_heads"], c["dim"], c["page"]
        out = torch.zeros(B, H, D, dtype=torch.float64, device="cuda")
        scores = s["scores"].double() if c["track"] else None
        for b, n in enumerate(s["lengths"].tolist()):
            if n == 0:
                continue
            pages = s["page_table"][b, : -(-n // page)].long()
            for j in range(N):
                def rows(codes, exps):
                    x = tab[codes[0, pages, j].reshape(-1, D)[:n].long() % tab.numel()]
                    return x if exps is None else x * torch.exp2(exps[0, pages, j].reshape(-1)[:n].double())[:, None]
                heads = slice(j * (H // N), (j + 1) * (H // N))
                t = s["q"][b, heads].double() @ rows(s["k"], s["k_exp"]).T / math.sqrt(D)
                p = torch.softmax(t, dim=-1)
                out[b, heads] = p @ rows(s["v"], s["v_exp"])
                if scores is not None:
                    scores[0, b, j, :n] += p.sum(0)
        return {"out": out, "scores": scores} if c["track"] else {"out": out}
    if c["op"] == "append":
        z = torch.view_as_complex(torch.stack(s["q"].double().chunk(2, dim=-1), dim=-1))
        at = s["positions"].long()
        z = z * torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None]
        return {"q": torch.cat((z.real, z.imag), dim=-1), "k": None, "v": None, "k_exp": None, "v_exp": None}
    # eviction: where the accumulated weights of the kept entries end up, row by row
    L, M = c["length"], c["budget"]
    pos, w, out = s["track"].cpu().numpy(), s["weights"].double().cpu().numpy(), s["scores"].double().cpu().numpy()
    for at in np.ndindex(pos.shape[:3]):
        p, key = pos[at][:L], w[at][:L].copy()
        key[(p < c["sinks"]) | (p > p.max() - c["recent"])] = np.inf
        best = np.sort(np.lexsort((np.arange(L), -key))[:M])
        front = best[best < M]
        holes = np.setdiff1d(np.arange(M), front, assume_unique=True)
        out[at][holes] = out[at][best[best >= M]]
    return {"keep": None, "k": None, "v": None, "k_exp": None, "v_exp": None, "scores": torch.from_numpy(out),
            "positions": None}
