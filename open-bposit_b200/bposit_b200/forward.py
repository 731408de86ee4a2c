"""A model-shaped forward around the W8A8 linear (the callers either side of the
hot path): a Qwen2.5-0.5B-shaped decoder stack with random-init weights
(seeded; there is no checkpoint).

Everything except the linears -- embedding, RMSNorm, RoPE, causal grouped-query
attention, SiLU gating -- runs in fp32 torch; every linear is a torch.nn.Linear
that ``bpositify`` turns into a BpositLinear (bp8 W8A8, exact quire, one
bposit32 round, nearest fp32 out).  q/k/v and gate/up are fused along N, which
is exact because GEMM outputs are column-independent.

Generating text goes through the paged b-posit key-value cache (``kv``):
``prefill`` runs a prompt batch and stores every layer's keys and values,
``step`` runs one token per sequence against the cache -- ``ops.kv_append``
rotates the queries and keys and writes the codes, ``ops.paged_attention``
reads them -- and ``generate`` alternates ``step`` with a greedy choice, evicting
the entries that were attended to least when the cache is given a budget.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

from . import ops
from .kv import PagedKVCache, protected
from .nn import bpositify

QWEN05 = dict(hidden=896, inter=4864, heads=14, kv_heads=2, head_dim=64, layers=24, vocab=151936,
              rope_theta=1e6, eps=1e-6)


class RMSNorm(torch.nn.Module):
    def __init__(self, dim: int, eps: float):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.ones(dim), requires_grad=False)
        self.eps = eps

    def forward(self, x):
        return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + self.eps) * self.weight


def _rope(x, cos, sin):
    x1, x2 = x[..., : x.shape[-1] // 2], x[..., x.shape[-1] // 2:]
    return x * cos + torch.cat((-x2, x1), dim=-1) * sin


class DecoderLayer(torch.nn.Module):
    def __init__(self, c):
        super().__init__()
        h, hd = c["hidden"], c["head_dim"]
        self.c = c
        self.ln1 = RMSNorm(h, c["eps"])
        self.qkv = torch.nn.Linear(h, (c["heads"] + 2 * c["kv_heads"]) * hd, bias=True)
        self.o = torch.nn.Linear(c["heads"] * hd, h, bias=False)
        self.ln2 = RMSNorm(h, c["eps"])
        self.gate_up = torch.nn.Linear(h, 2 * c["inter"], bias=False)
        self.down = torch.nn.Linear(c["inter"], h, bias=False)

    def forward(self, x, cos, sin, store=None):
        """`store(k, v)`, if given, receives the layer's rotated keys and its
        values, [B, kv_heads, S, head_dim]."""
        c = self.c
        B, S, _ = x.shape
        hd, nh, nkv = c["head_dim"], c["heads"], c["kv_heads"]
        qkv = self.qkv(self.ln1(x))
        q, k, v = qkv.split([nh * hd, nkv * hd, nkv * hd], dim=-1)
        q = _rope(q.view(B, S, nh, hd).transpose(1, 2), cos, sin)
        k = _rope(k.view(B, S, nkv, hd).transpose(1, 2), cos, sin)
        v = v.view(B, S, nkv, hd).transpose(1, 2)
        if store is not None:
            store(k, v)
        rep = nh // nkv
        a = F.scaled_dot_product_attention(q, k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1),
                                           is_causal=True)
        x = x + self.o(a.transpose(1, 2).reshape(B, S, nh * hd))
        g, u = self.gate_up(self.ln2(x)).chunk(2, dim=-1)
        return x + self.down(F.silu(g) * u)

    def step(self, x, cache, layer: int, cos, sin, positions):
        """One token per sequence, x [B, hidden], against `cache`, which has
        room for it (PagedKVCache.advance); cos, sin: the tables of all
        positions, positions [B] int32."""
        c = self.c
        B = x.shape[0]
        hd, nh, nkv = c["head_dim"], c["heads"], c["kv_heads"]
        qkv = self.qkv(self.ln1(x)).view(B, nh + 2 * nkv, hd)
        q, k, v = qkv.split([nh, nkv, nkv], dim=1)
        q = ops.kv_append(cache, k, v, q=q, cos=cos, sin=sin, positions=positions, layer=layer)
        a = ops.paged_attention(cache, q, layer=layer, max_length=cache.bound, accumulate=cache.scores is not None)
        x = x + self.o(a.reshape(B, nh * hd))
        g, u = self.gate_up(self.ln2(x)).chunk(2, dim=-1)
        return x + self.down(F.silu(g) * u)


class QwenShaped(torch.nn.Module):
    """Qwen2.5-0.5B-shaped decoder stack (no LM head): token ids -> final hidden."""

    def __init__(self, c=None, layers: int | None = None):
        super().__init__()
        c = dict(QWEN05 if c is None else c)
        if layers is not None:
            c["layers"] = layers
        self.c = c
        self.embed = torch.nn.Embedding(c["vocab"], c["hidden"])
        self.layers = torch.nn.ModuleList([DecoderLayer(c) for _ in range(c["layers"])])
        self.norm = RMSNorm(c["hidden"], c["eps"])

    @torch.no_grad()
    def init_weights(self, seed: int = 0):
        dev = self.embed.weight.device
        g = torch.Generator(device=dev).manual_seed(seed)
        for p in self.parameters():          # matrices N(0, 0.02^2); RMSNorm weights stay 1
            if p.dim() >= 2:
                p.copy_(torch.randn(p.shape, generator=g, device=dev) * 0.02)
        for layer in self.layers:
            layer.qkv.bias.copy_(torch.randn(layer.qkv.bias.shape, generator=g, device=dev) * 0.02)
        return self

    def linear_ops(self, tokens: int) -> float:
        """2 * tokens * sum(N * K) over the decoder linears."""
        n = 0
        for layer in self.layers:
            for lin in (layer.qkv, layer.o, layer.gate_up, layer.down):
                n += lin.in_features * lin.out_features
        return 2.0 * tokens * n

    @torch.no_grad()
    def forward(self, ids):
        c = self.c
        S = ids.shape[1]
        x = self.embed(ids)
        pos = torch.arange(S, device=ids.device, dtype=torch.float32)
        inv = 1.0 / (c["rope_theta"] ** (torch.arange(0, c["head_dim"], 2, device=ids.device,
                                                         dtype=torch.float32) / c["head_dim"]))
        ang = torch.outer(pos, inv)
        cos = torch.cat((ang.cos(), ang.cos()), -1)[None, None]
        sin = torch.cat((ang.sin(), ang.sin()), -1)[None, None]
        for layer in self.layers:
            x = layer(x, cos, sin)
        return self.norm(x)

    # ---- generation ----
    def rope_tables(self, rows: int):
        """cos, sin [rows, head_dim / 2] float32, the values that forward uses."""
        c = self.c
        dev = self.embed.weight.device
        pos = torch.arange(rows, device=dev, dtype=torch.float32)
        inv = 1.0 / (c["rope_theta"] ** (torch.arange(0, c["head_dim"], 2, device=dev,
                                                      dtype=torch.float32) / c["head_dim"]))
        ang = torch.outer(pos, inv)
        return ang.cos(), ang.sin()

    def new_cache(self, batch: int, max_tokens: int, fmt="bp8", page_size: int = 64, track: bool = False):
        """An empty PagedKVCache of this model's shape."""
        c = self.c
        return PagedKVCache(batch, c["kv_heads"], c["head_dim"], max_tokens, layers=c["layers"], fmt=fmt,
                            page_size=page_size, track=track, device=self.embed.weight.device)

    def _check_cache(self, cache):
        """Refuses a cache that the layers cannot use, before its lengths move."""
        c = self.c
        if (cache.kv_heads, cache.head_dim) != (c["kv_heads"], c["head_dim"]) or cache.layers < c["layers"]:
            raise ValueError(f"the cache has {cache.layers} layers of {cache.kv_heads} heads of {cache.head_dim}, the "
                             f"model {c['layers']} of {c['kv_heads']} of {c['head_dim']}")

    @torch.no_grad()
    def prefill(self, ids, cache, lengths=None):
        """The forward of prompts ids [B, S] (padded on the right to S when
        `lengths`, one int per prompt, is given) whose keys and values also
        enter the empty `cache`.  Returns forward(ids)."""
        B, S = ids.shape
        dev = ids.device
        self._check_cache(cache)
        if B != cache.batch or not cache.is_empty():
            raise ValueError("prefill needs an empty cache of the batch's size")
        n = [S] * B if lengths is None else [int(x) for x in lengths]
        if len(n) != B or min(n) < 0 or max(n) > S:
            raise ValueError(f"lengths must be {B} numbers from 0 to {S}")
        cache.advance(torch.tensor(n, dtype=torch.int32, device=dev), most=max(n))
        places = torch.arange(S, dtype=torch.int32, device=dev).repeat(B)
        seqs = torch.arange(B, dtype=torch.int32, device=dev).repeat_interleave(S)
        if lengths is not None:          # padding is not stored
            seqs = torch.where(places < cache.lengths.repeat_interleave(S), seqs, -1).to(torch.int32)
        c = self.c
        shape = (B * S, c["kv_heads"], c["head_dim"])
        cos, sin = (torch.cat((t, t), -1)[None, None] for t in self.rope_tables(S))
        x = self.embed(ids)
        for i, layer in enumerate(self.layers):
            x = layer(x, cos, sin, store=lambda k, v: ops.kv_append(
                cache, k.transpose(1, 2).reshape(shape), v.transpose(1, 2).reshape(shape), seqs=seqs, places=places,
                layer=i))
        return self.norm(x)

    @torch.no_grad()
    def step(self, ids, cache, tables):
        """The next token of every sequence, ids [B]: its final hidden state
        [B, hidden], its keys and values appended to `cache`.  tables:
        rope_tables of at least the tokens that the sequences will have seen.
        May be captured into a graph: each replay is one step further."""
        self._check_cache(cache)
        if ids.shape != (cache.batch,):
            raise ValueError(f"ids must be one token for each of the cache's {cache.batch} sequences, got "
                             f"{list(ids.shape)}")
        if cache.seen is None:
            raise ValueError("a cache over the caller's tensors does not count the tokens seen, the positions")
        cache.advance()
        positions = cache.seen - 1
        x = self.embed(ids)
        for i, layer in enumerate(self.layers):
            x = layer.step(x, cache, i, *tables, positions)
        return self.norm(x)

    def logits(self, hidden):
        """Logits over the vocabulary (tied embedding)."""
        return F.linear(hidden, self.embed.weight)

    @torch.no_grad()
    def generate(self, ids, new_tokens: int, lengths=None, fmt="bp8", page_size: int = 64, budget: int | None = None,
                 recent: int | None = None, sinks: int | None = None):
        """Greedy continuation of prompts ids [B, S]: [B, new_tokens] token ids.
        With `budget` the cache of every layer and kv head is cut down to that
        many entries whenever a page more has been filled: the `sinks` first and
        `recent` last ones (default 4 and 64, fewer in a budget that does not hold
        them) and, of the others, those that the new tokens attended to most."""
        if new_tokens < 1:
            raise ValueError("new_tokens must be positive")
        B, S = ids.shape
        if S < 1 or (lengths is not None and min(int(x) for x in lengths) < 1):
            raise ValueError("prompts have at least one token")
        if budget is not None:
            recent, sinks = protected(budget, recent, sinks)
        cache = self.new_cache(B, S + new_tokens if budget is None else max(S, budget + page_size) + 1, fmt, page_size,
                               track=budget is not None)
        tables = self.rope_tables(S + new_tokens)
        hidden = self.prefill(ids, cache, lengths)
        last = (torch.full((B,), S, device=ids.device) if lengths is None else
                torch.as_tensor(lengths, device=ids.device)).long() - 1
        token = self.logits(hidden[torch.arange(B, device=ids.device), last.clamp(min=0)]).argmax(-1)
        out = [token]
        for _ in range(new_tokens - 1):
            token = self.logits(self.step(token, cache, tables)).argmax(-1)
            out.append(token)
            if budget is not None and cache.longest >= budget + page_size:
                cache.evict(budget, recent=recent, sinks=sinks)
        return torch.stack(out, dim=1)


def qwen05(layers: int = 24, device="cuda", seed: int = 0, bposit: bool = True) -> QwenShaped:
    m = QwenShaped(layers=layers).to(device).init_weights(seed)
    return bpositify(m) if bposit else m


def synthetic_ids(batch: int, seq: int, vocab: int = QWEN05["vocab"], seed: int = 0, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    return torch.randint(0, vocab, (batch, seq), generator=g, device=device)
