"""Plain 64-bit forms of the paged key-value cache's operators, for the tests."""
from __future__ import annotations

import math

import numpy as np
import torch


def code_values(orc, fmt: str) -> torch.Tensor:
    """float64 value of every code (zero and NaR: 0)."""
    n, bits = (256, 8) if fmt == "bp8" else (65536, 16)
    return torch.from_numpy(orc.decode_f32(np.arange(n).astype(np.uint8 if bits == 8 else np.uint16), bits)
                            .astype(np.float64))


def held(cache, table, which: str, layer: int, b: int, hk: int, n: int) -> torch.Tensor:
    """float64 rows [n, head_dim] that a sequence's first n entries hold (CPU)."""
    pages = cache.page_table[b, : -(-n // cache.page_size)].long().cpu()
    pool = getattr(cache, which)[layer].cpu()
    pool = pool if pool.dtype == torch.uint8 else pool.view(torch.int16)
    codes = pool[pages, hk].reshape(-1, cache.head_dim)[:n].long() % table.numel()
    x = table[codes]
    e = getattr(cache, which + "_exp")
    return x if e is None else torch.ldexp(x, e[layer].cpu()[pages, hk].reshape(-1)[:n].int()[:, None])


def attention(cache, table, q: torch.Tensor, layer: int = 0, scale=None, lengths=None):
    """(out, lse, weights {(b, hk): [n] sums}, bound) in float64; `bound` is the
    derived error of an fp32 evaluation, per output (see below)."""
    B, H, D = q.shape
    G = H // cache.kv_heads
    scale = D ** -0.5 if scale is None else scale
    lens = cache.lengths.tolist() if lengths is None else lengths
    out = torch.zeros(B, H, D, dtype=torch.float64)
    bound = torch.zeros(B, H, D, dtype=torch.float64)
    lse = torch.full((B, H), -math.inf, dtype=torch.float64)
    lse_bound = torch.zeros(B, H, dtype=torch.float64)
    weights, u = {}, 2.0 ** -24
    for b, n in enumerate(lens):
        n = max(0, min(n, cache.capacity))
        if n == 0:
            continue
        for hk in range(cache.kv_heads):
            k, v = (held(cache, table, w, layer, b, hk, n) for w in ("k", "v"))
            x = q[b, hk * G:(hk + 1) * G].double().cpu()
            s = x @ k.T * scale
            p = torch.softmax(s, dim=-1)
            h = slice(hk * G, (hk + 1) * G)
            out[b, h], lse[b, h] = p @ v, torch.logsumexp(s, dim=-1)
            weights[b, hk] = p.sum(0)
            # a score: D exact products summed in fp32 (each addition off by a step, 2u, at most: the tensor
            # cores truncate), then scaled three times; both it and the maximum enter the exponential, whose
            # own error is two steps; sums of weights and of weighted values add a tile of 64 entries (up to
            # three terms each), then tiles, then parts of the cache's length
            ds = 2 * u * (D + 8) * (x.abs() @ k.abs().T * scale).amax(-1) + u * s.abs().amax(-1) * 4
            rel = 2 * ds + u * (400 + n / 32)
            bound[b, h] = 2 * rel[:, None] * (p @ v.abs())
            lse_bound[b, h] = rel + 4 * u * lse[b, h].abs()
            weights[b, hk, "bound"] = (2 * rel[:, None] * p).sum(0)
    return out, lse, weights, bound, lse_bound


def rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x [tokens, heads, D] rotated by rows cos, sin [tokens, D/2], float64 rounded to fp32 (CPU)."""
    a, b = x.double().cpu().chunk(2, dim=-1)
    c, s = cos.double().cpu()[:, None], sin.double().cpu()[:, None]
    return torch.cat((a * c - b * s, b * c + a * s), dim=-1).float()


def rotated_queries(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor):
    """(rotation of x in float64, bound of an fp32 product and fma and the rounding to x's type)."""
    a, b = x.double().cpu().chunk(2, dim=-1)
    c, s = cos.double().cpu()[:, None], sin.double().cpu()[:, None]
    y = torch.cat((a * c - b * s, b * c + a * s), dim=-1)
    u, step = 2.0 ** -24, {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[x.dtype]
    inner = u * torch.cat(((b * s).abs(), (a * s).abs()), dim=-1)      # the product that is rounded first
    outer = inner + u * (y.abs() + inner)                              # the fma's own rounding
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 2.0 ** -148     # half a step of the smallest numbers
    return y, outer + step * (y.abs() + outer) + tiny


def encode(orc, x: torch.Tensor, fmt: str):
    """Codes (numpy) and exponents (numpy int8 or None) of fp32 rows."""
    a = x.numpy()
    if fmt == "bp16":
        return orc.encode_bp16(a.reshape(-1)).reshape(a.shape), None
    top = np.where(np.isfinite(a), np.abs(a), 0).max(-1).astype(np.float64)
    e = np.where(top > 0, np.maximum(np.frexp(top)[1] - 4, -126), 0)
    c = orc.quantize_bp8_f64(np.ldexp(a.astype(np.float64), -e[..., None]).reshape(-1), nearest=True)
    c = np.where(np.isnan(a.reshape(-1)), 0x80, c)
    return c.reshape(a.shape).astype(np.uint8), e.astype(np.int8)


def evict_keep(pos: np.ndarray, w: np.ndarray, n: int, budget: int, recent: int, sinks: int) -> np.ndarray:
    """The keep list of one row."""
    if n <= budget:
        return np.where(np.arange(budget) < n, np.arange(budget), -1)
    p, key = pos[:n].astype(np.int64), w[:n].astype(np.float64)
    key = np.where(np.isnan(key), -np.inf, key)
    key[(p < sinks) | (p > p.max() - recent)] = np.inf
    # NaN is behind -inf: the second key tells them apart
    behind = np.isnan(w[:n]) & (key == -np.inf)
    best = np.sort(np.lexsort((np.arange(n), behind, -key))[:budget])
    keep = np.arange(budget)
    holes = np.setdiff1d(keep, best)
    keep[holes] = best[best >= budget]
    return keep
