"""The paged key-value cache without a GPU: the row encoder against the oracle, and
every refusal of the C entry points and of the Python layer."""
from __future__ import annotations

import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

from conftest import REPO


@pytest.fixture(scope="module")
def host():
    build = os.path.join(REPO, "tests", "_build")
    os.makedirs(build, exist_ok=True)
    so = os.path.join(build, "host_kv_check.so")
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-o", so,
                    os.path.join(REPO, "tests", "host_kv_check.cpp")], check=True)
    return ctypes.CDLL(so)


@pytest.mark.parametrize("e", [0, -3, 4, 24, -24, 100, -100, 124, -126])
def test_row_encoder_matches_oracle(host, orc, e):
    """bp8_encode_exp(x, e) is the oracle's round-to-nearest bp8 of x / 2^e in float64."""
    u = np.arange(0, 1 << 32, 4099, dtype=np.uint64).astype(np.uint32)
    # around every value and midpoint that the format has at this exponent
    g = orc.decode_f32(np.arange(1, 128).astype(np.uint8), 8).astype(np.float64)
    m = np.concatenate((g, (g[1:] + g[:-1]) / 2)) * 2.0 ** e
    m = m[(m < 3e38) & (m > 1e-45)].astype(np.float32).view(np.uint32)
    u = np.concatenate((u, m, m - 1, m + 1, (m + 1) | np.uint32(1 << 31),
                        np.array([0, 1 << 31, 1, 0x7F800000, 0xFF800000, 0x7FC00000, 0x7F7FFFFF], np.uint32)))
    u = np.ascontiguousarray(u)
    out = np.empty(u.size, np.uint8)
    host.kv_encode_bp8(u.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(u.size), e,
                       out.ctypes.data_as(ctypes.c_void_p))
    with np.errstate(invalid="ignore"):
        x = u.view(np.float32).astype(np.float64)
    ref = np.where(np.isnan(x), 0x80, orc.quantize_bp8_f64(np.ldexp(x, -e), nearest=True)).astype(np.uint8)
    assert np.array_equal(out, ref)


@pytest.mark.parametrize("fmt", [8, 16])
def test_closed_form_encoders_match_oracle(host, orc, fmt):
    """The encoders without cases, on a sweep of all patterns and on every binade's ties and edges."""
    top = (np.arange(512, dtype=np.uint64) << 23)[:, None]
    low = np.concatenate([[0, 1, 0x7FFFFF, 0x7FFFFE, 0x400000, 0x3FFFFF, 0x400001],
                          *[(np.array([1, 3, 5, 7]) << b) + d for b in range(10, 23) for d in (-1, 0, 1)]])
    u = np.concatenate((np.arange(0, 1 << 32, 1021, dtype=np.uint64), (top + (low & 0x7FFFFF)[None]).reshape(-1)))
    u = np.ascontiguousarray(u.astype(np.uint32))
    out = np.empty(u.size, np.uint32)
    host.kv_encode_near(u.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(u.size), fmt,
                        out.ctypes.data_as(ctypes.c_void_p))
    with np.errstate(invalid="ignore"):
        x = u.view(np.float32)
        ref = orc.quantize_bp8(x) if fmt == 8 else orc.encode_bp16(x)
    ref = ref[0] if isinstance(ref, tuple) else ref
    assert np.array_equal(out, ref.astype(np.uint32))


def test_floor_log2(host):
    a = np.concatenate((np.arange(1, 0x7F800000, 65521), np.arange(1, 70000), [0x007FFFFF, 0x00800000])).astype(np.uint32)
    out = np.empty(a.size, np.int32)
    host.kv_floor_log2(a.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(a.size), out.ctypes.data_as(ctypes.c_void_p))
    assert np.array_equal(out, np.frexp(a.view(np.float32).astype(np.float64))[1] - 1)


# ---- the C entry points: everything below is refused before any device work ----
def struct(**kw):
    from bposit_b200.kv import _Struct
    d = dict(fmt=8, layers=2, pages=8, page_size=16, kv_heads=2, head_dim=64, batch=2, max_pages=4, k=4096, v=8192,
             k_exp=16, v_exp=32, page_table=4, lengths=4, positions=4, scores=4)
    d.update(kw)
    return _Struct(**d)


BAD_CACHE = [(dict(fmt=9), "FMT"), (dict(fmt=16), "EINVAL"), (dict(head_dim=48), "ERANGE"), (dict(head_dim=256), "ERANGE"),
             (dict(page_size=8), "ERANGE"), (dict(page_size=48), "ERANGE"), (dict(page_size=2048), "ERANGE"),
             (dict(layers=0), "EINVAL"), (dict(kv_heads=0), "EINVAL"), (dict(pages=-1), "EINVAL"),
             (dict(batch=5000), "ERANGE"), (dict(kv_heads=2000), "ERANGE"), (dict(max_pages=1 << 27), "ERANGE"),
             (dict(k=None), "EINVAL"), (dict(v=None), "EINVAL"), (dict(k_exp=None), "EINVAL"),
             (dict(lengths=None), "EINVAL"), (dict(page_table=None), "EINVAL"), (dict(k=4100), "EALIGN"),
             (dict(v_exp=33), "EALIGN")]


def code(name):
    from bposit_b200 import _lib
    return getattr(_lib, "BP_EFMT" if name == "FMT" else "BP_" + name)


def append(L, c, layer=0, dtype=0, tokens=2, k=16, ks=128, v=16, vs=128, q=16, heads=4, qs=256, cos=16, sin=16,
           rows=10, positions=None, seqs=None, places=None, q_out=16):
    return L.bp_kv_append(ctypes.byref(c) if c else None, layer, dtype, tokens, k, ks, v, vs, q, heads, qs, cos, sin,
                          rows, positions, seqs, places, q_out, None)


def attend(L, c, layer=0, dtype=0, heads=4, q=16, qs=256, out=16, lse=None, scale=1.0, most=0, acc=0, ws=None, n=0):
    return L.bp_paged_attention(ctypes.byref(c) if c else None, layer, dtype, heads, q, qs, out, lse, scale, most, acc,
                                ws, n, None)


def evict(L, c, w=None, budget=4, recent=0, sinks=0, keep=None):
    return L.bp_kv_evict(ctypes.byref(c) if c else None, w, budget, recent, sinks, keep, None)


@pytest.mark.parametrize("kw,want", BAD_CACHE)
def test_bad_caches_are_refused(kw, want):
    from bposit_b200 import _lib
    L = _lib.lib()
    for call in (append, attend, evict):
        assert call(L, struct(**kw)) == code(want), (call.__name__, L.bp_last_error())
        assert call(L, None) == _lib.BP_EINVAL


@pytest.mark.parametrize("kw,want", [
    (dict(layer=2), "EINVAL"), (dict(layer=-1), "EINVAL"), (dict(dtype=3), "FMT"), (dict(tokens=-1), "EINVAL"),
    (dict(tokens=3), "EINVAL"), (dict(seqs=16), "EINVAL"), (dict(places=16), "EINVAL"), (dict(cos=None), "EINVAL"),
    (dict(sin=None), "EINVAL"), (dict(rows=0), "EINVAL"), (dict(heads=0), "EINVAL"), (dict(k=None), "EINVAL"),
    (dict(v=None), "EINVAL"), (dict(q_out=None), "EINVAL"), (dict(ks=64), "EINVAL"), (dict(qs=252), "EINVAL"),
    (dict(ks=130), "EALIGN"), (dict(dtype=1, vs=132), "EALIGN"), (dict(q=24), "EALIGN"), (dict(cos=20), "EALIGN"),
    (dict(cos=None, sin=None, rows=0), "EINVAL")])
def test_append_refusals(kw, want):
    from bposit_b200 import _lib
    L = _lib.lib()
    assert append(L, struct(), **kw) == code(want), L.bp_last_error()


@pytest.mark.parametrize("kw,want", [
    (dict(layer=2), "EINVAL"), (dict(dtype=-1), "FMT"), (dict(heads=3), "EINVAL"), (dict(heads=0), "EINVAL"),
    (dict(q=None), "EINVAL"), (dict(out=None), "EINVAL"), (dict(qs=255), "EINVAL"), (dict(qs=258), "EALIGN"),
    (dict(out=8), "EALIGN"), (dict(most=-1), "EINVAL"), (dict(ws=128, n=1 << 30), "EALIGN"),
    (dict(acc=1, ws=256, n=1), "EWORKSPACE")])
def test_attention_refusals(kw, want):
    from bposit_b200 import _lib
    L = _lib.lib()
    assert attend(L, struct(), **kw) == code(want), L.bp_last_error()


def test_attention_without_scores_is_refused():
    from bposit_b200 import _lib
    L = _lib.lib()
    assert attend(L, struct(scores=None), acc=1) == _lib.BP_EINVAL
    assert L.bp_paged_attention_workspace_size(ctypes.byref(struct(scores=None)), 4, 0, 1) == 0
    assert L.bp_paged_attention_workspace_size(ctypes.byref(struct()), 3, 0, 0) == 0
    assert L.bp_paged_attention_workspace_size(ctypes.byref(struct()), 4, 0, 1) > 0


@pytest.mark.parametrize("kw", [dict(budget=0), dict(recent=-1), dict(sinks=-1)])
def test_evict_refusals(kw):
    from bposit_b200 import _lib
    L = _lib.lib()
    assert evict(L, struct(), **kw) == _lib.BP_EINVAL
    assert evict(L, struct(positions=None)) == _lib.BP_EINVAL
    assert evict(L, struct(scores=None)) == _lib.BP_EINVAL


def test_empty_calls_succeed_without_a_device():
    from bposit_b200 import _lib
    L = _lib.lib()
    none = struct(batch=0)
    assert append(L, none, tokens=0) == 0 and attend(L, none) == 0 and evict(L, none) == 0
    assert append(L, struct(), tokens=0, seqs=16, places=16) == 0
    assert append(L, struct(), tokens=0, q=None, heads=0) == 0


# ---- the Python layer ----
def tensors(fmt="bp8", **kw):
    L, P, H, S, D, B, M = 2, 8, 2, 16, 64, 2, 4
    dt = torch.uint8 if fmt == "bp8" else torch.int16
    d = dict(k=torch.zeros(L, P, H, S, D, dtype=dt), v=torch.zeros(L, P, H, S, D, dtype=dt),
             page_table=torch.zeros(B, M, dtype=torch.int32), lengths=torch.zeros(B, dtype=torch.int32))
    if fmt == "bp8":
        d.update(k_exp=torch.zeros(L, P, H, S, dtype=torch.int8), v_exp=torch.zeros(L, P, H, S, dtype=torch.int8))
    else:
        d.update(k=d["k"].view(torch.uint16), v=d["v"].view(torch.uint16))
    d.update(kw)
    return d


@pytest.mark.parametrize("kw,match", [
    (dict(), "CUDA"), (dict(k_exp=None), "k_exp"), (dict(v=torch.zeros(2, 8, 2, 16, 32, dtype=torch.uint8)), "v must"),
    (dict(k=torch.zeros(8, 2, 16, 64, dtype=torch.uint8)), "k must"),
    (dict(k=torch.zeros(2, 8, 2, 16, 64)), "k must"),
    (dict(k=torch.zeros(2, 8, 2, 16, 48, dtype=torch.uint8)), "head_dim"),
    (dict(k=torch.zeros(2, 8, 2, 24, 64, dtype=torch.uint8)), "page_size"),
    (dict(page_table=torch.zeros(2, 4, dtype=torch.int64)), "page_table"),
    (dict(page_table=torch.zeros(8, dtype=torch.int32)), "page_table"),
    (dict(page_table=torch.zeros(4, 2, dtype=torch.int32).t()), "page_table"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths"),
    (dict(lengths=torch.zeros(2, 2, dtype=torch.int32)), "lengths"),
    (dict(positions=torch.zeros(2, 2, 2, 63, dtype=torch.int32)), "positions"),
    (dict(scores=torch.zeros(2, 2, 2, 64, dtype=torch.float64)), "scores")])
def test_cache_tensors_are_checked(kw, match):
    from bposit_b200.kv import PagedKVCache
    with pytest.raises(ValueError, match=match):
        PagedKVCache.over(**tensors(**kw))


def test_bp16_cache_takes_no_exponents():
    from bposit_b200.kv import PagedKVCache
    with pytest.raises(ValueError, match="CUDA"):
        PagedKVCache.over(**tensors("bp16"))
    with pytest.raises(ValueError, match="neither"):
        PagedKVCache.over(**tensors("bp16", k_exp=torch.zeros(2, 8, 2, 16, dtype=torch.int8)))
    with pytest.raises(KeyError):
        PagedKVCache(1, 1, 64, 16, fmt="bp4", device="cpu")
    with pytest.raises(ValueError):
        PagedKVCache(0, 1, 64, 16, device="cpu")
