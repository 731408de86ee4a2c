"""Paged key-value cache in b-posit codes, for generating text with a model whose
linears are b-posit GEMMs.

    cache = PagedKVCache(batch=8, kv_heads=2, head_dim=64, max_tokens=4096, layers=24)
    cache.advance()                                   # room for one token per sequence
    for i, layer in enumerate(layers):
        q = ops.kv_append(cache, k, v, q=q, cos=cos, sin=sin, positions=pos, layer=i)
        out = ops.paged_attention(cache, q, layer=i)

Keys and values are bp8 codes with one power-of-two exponent per (token, kv
head) -- 65 bytes for a 64-wide head against 256 in fp32 -- or bp16 codes.  The
pools are [layers, pages, kv_heads, page_size, head_dim]; ``page_table`` [batch,
max_pages] names the pages of each sequence and ``lengths`` [batch] its entries,
both int32 on the device and shared by all layers.  With ``track=True`` the cache
also keeps, per (layer, sequence, kv head), the rotary position of every entry
and the attention weight it has received (``ops.paged_attention(...,
accumulate=True)``); ``evict`` keeps the entries that were attended to most.
Tables, lengths and pools may be written by the caller at any time, on the
stream that the ops run on; whoever makes a sequence longer than ``longest``, the
host's bound of the lengths, sets that too.
"""
from __future__ import annotations

import ctypes

import torch

from . import ops


class _Struct(ctypes.Structure):
    """bp_kv_cache of the C ABI."""
    _fields_ = [(n, ctypes.c_int32) for n in ("fmt", "layers", "pages", "page_size", "kv_heads", "head_dim",
                                              "batch", "max_pages")] + \
               [(n, ctypes.c_void_p) for n in ("k", "v", "k_exp", "v_exp", "page_table", "lengths", "positions",
                                               "scores")]


def protected(budget: int, recent: int | None = None, sinks: int | None = None) -> tuple[int, int]:
    """(recent, sinks) for evictions to `budget` entries, checked or chosen: the
    4 first and 64 last tokens, fewer where the budget does not hold them.  More
    than `budget` of them would compete by place, and the newest would go."""
    if budget < 1:
        raise ValueError("budget must be positive")
    if sinks is None:
        sinks = min(4, budget // 2 if recent is None else max(0, budget - recent))
    if recent is None:
        recent = min(64, budget - sinks)
    if min(recent, sinks) < 0 or recent + sinks > budget:
        raise ValueError(f"a budget of {budget} entries does not hold the {sinks} first and {recent} last tokens")
    return recent, sinks


_TENSORS = ("k", "v", "k_exp", "v_exp", "page_table", "lengths", "positions", "scores")


class PagedKVCache:
    """See the module docstring.  ``max_tokens`` is each sequence's capacity,
    rounded up to whole pages; every sequence gets its own pages."""

    def __init__(self, batch: int, kv_heads: int, head_dim: int, max_tokens: int, *, layers: int = 1, fmt="bp8",
                 page_size: int = 64, track: bool = False, device="cuda"):
        f = ops.fmt_bits(fmt)
        if min(batch, kv_heads, max_tokens, layers) < 1:
            raise ValueError("batch, kv_heads, max_tokens and layers must be positive")
        if page_size < 1:
            raise ValueError("page_size must be positive")
        per = -(-max_tokens // page_size)
        shape = (layers, batch * per, kv_heads, page_size)
        dt = torch.uint8 if f == 8 else torch.uint16
        k, v = (torch.zeros(shape + (head_dim,), dtype=dt, device=device) for _ in range(2))
        ke = ve = pos = scores = None
        if f == 8:
            ke, ve = (torch.zeros(shape, dtype=torch.int8, device=device) for _ in range(2))
        if track:
            pos = torch.zeros((layers, batch, kv_heads, per * page_size), dtype=torch.int32, device=device)
            scores = torch.zeros(pos.shape, dtype=torch.float32, device=device)
        table = torch.arange(batch * per, dtype=torch.int32, device=device).view(batch, per)
        self._set(k, v, table, torch.zeros(2, batch, dtype=torch.int32, device=device), ke, ve, pos, scores)
        self.longest = 0

    @classmethod
    def over(cls, k, v, page_table, lengths, *, k_exp=None, v_exp=None, positions=None, scores=None):
        """A cache over the caller's own tensors: k, v [layers, pages, kv_heads,
        page_size, head_dim] uint8 (bp8, with k_exp, v_exp [layers, pages,
        kv_heads, page_size] int8) or uint16 (bp16); page_table [batch,
        max_pages] and lengths [batch] int32; positions int32 and scores float32
        [layers, batch, kv_heads, max_pages * page_size].  Nothing is copied.
        ``longest``, the host's bound of the lengths, starts at the capacity; set
        it to what the lengths really are, or ``advance`` has to look.  Such a
        cache does not count the tokens seen (``seen`` is None): whoever appends to
        it gives the positions."""
        c = cls.__new__(cls)
        if not isinstance(lengths, torch.Tensor) or lengths.dim() != 1:
            raise ValueError("lengths must be a [batch] int32 tensor")
        c._set(k, v, page_table, lengths, k_exp, v_exp, positions, scores)
        c.longest = c.capacity
        return c

    def _set(self, k, v, table, lengths, k_exp, v_exp, positions, scores):
        if not isinstance(k, torch.Tensor) or k.dim() != 5 or k.dtype not in (torch.uint8, torch.uint16):
            raise ValueError("k must be a [layers, pages, kv_heads, page_size, head_dim] uint8 or uint16 tensor")
        layers, pages, heads, page, dim = k.shape
        bp8 = k.dtype == torch.uint8
        if dim not in (32, 64, 96, 128):
            raise ValueError(f"head_dim must be 32, 64, 96 or 128, got {dim}")
        if not 16 <= page <= 1024 or page & (page - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page}")
        if (k_exp is None) == bp8 or (v_exp is None) == bp8:
            raise ValueError("bp8 (uint8) caches have k_exp and v_exp, bp16 (uint16) caches have neither")
        if not isinstance(table, torch.Tensor) or table.dim() != 2:
            raise ValueError("page_table must be a [batch, max_pages] int32 tensor")
        batch, per = table.shape
        if batch > 2048:
            raise ValueError(f"batch of at most 2048 sequences, got {batch}")
        row = tuple(k.shape[:-1])
        track = (layers, batch, heads, per * page)
        lens = (2, batch) if lengths.dim() == 2 else (batch,)
        for name, t, dt, shape in (("k", k, k.dtype, tuple(k.shape)), ("v", v, k.dtype, tuple(k.shape)),
                                   ("k_exp", k_exp, torch.int8, row), ("v_exp", v_exp, torch.int8, row),
                                   ("page_table", table, torch.int32, (batch, per)),
                                   ("lengths", lengths, torch.int32, lens),
                                   ("positions", positions, torch.int32, track),
                                   ("scores", scores, torch.float32, track)):
            if t is None and name in ("k_exp", "v_exp", "positions", "scores"):
                continue
            if not isinstance(t, torch.Tensor) or t.dtype != dt or tuple(t.shape) != shape or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous {dt} tensor of shape {list(shape)}")
        for t in (k, v, k_exp, v_exp, table, lengths, positions, scores):
            if t is not None and (not t.is_cuda or t.device != k.device):
                raise ValueError("the cache's tensors must be CUDA tensors on one device")
        self.fmt = "bp8" if bp8 else "bp16"
        self.layers, self.pages, self.kv_heads, self.page_size, self.head_dim = layers, pages, heads, page, dim
        self.batch, self.max_pages, self.capacity, self.device = batch, per, per * page, k.device
        self.k, self.v, self.k_exp, self.v_exp = k, v, k_exp, v_exp
        self.page_table, self.positions, self.scores = table, positions, scores
        # [2, batch]: entries held, and tokens seen (they differ once entries were evicted)
        self._counts = lengths if lengths.dim() == 2 else None
        self.lengths = lengths if self._counts is None else lengths[0]
        self.seen = None if self._counts is None else lengths[1]
        ptr = lambda t: None if t is None else t.data_ptr()   # noqa: E731
        self._struct = _Struct(8 if bp8 else 16, layers, pages, page, heads, dim, batch, per, ptr(k), ptr(v),
                               ptr(k_exp), ptr(v_exp), ptr(table), ptr(self.lengths), ptr(positions), ptr(scores))
        self._ref = ctypes.byref(self._struct)
        self._replayed = False   # a change of the lengths was captured
        self._workspace = {}     # bytes that paged_attention needs, by its arguments

    def __setattr__(self, name, value):
        # the kernels are given the addresses of the tensors that the cache was made of
        if name in _TENSORS and name in self.__dict__:
            raise AttributeError(f"write into {name} in place, or make another cache over the tensors")
        super().__setattr__(name, value)

    def advance(self, n=1, most: int | None = None):
        """Make room for n more entries in every sequence (an int), or for n[b]
        in sequence b (an int32 tensor of which no value is above `most`); they
        are written by ``ops.kv_append`` in every layer.  Refused where they do
        not fit.  ``longest`` follows on the host as a bound of all lengths; the
        lengths themselves are read from the device (the host waits for it) only
        where that bound says that the entries do not fit, or cannot be trusted
        since such a call was captured.  Replays of a captured call are not
        refused: entries that they put past the capacity are dropped."""
        if not isinstance(n, int) and most is None:
            raise ValueError("give `most`, a bound of the counts that the host knows")
        more = n if isinstance(n, int) else int(most)
        if more < 0:
            raise ValueError("counts of new entries are not negative")
        longest = self.longest + more
        never = more > self.capacity and isinstance(n, int)
        if torch.cuda.is_current_stream_capturing():
            if self._replayed and not never:     # an earlier capture was counted, though it moved nothing
                longest = min(longest, self.capacity)
        elif (longest > self.capacity or self._replayed) and not never:
            longest = self._longest_held(n)
        if longest > self.capacity:
            raise ValueError(f"{longest} entries do not fit a capacity of {self.capacity}")
        self._note_capture()
        (self.lengths if self._counts is None else self._counts).add_(n)
        self.longest = longest

    def _longest_held(self, n=0) -> int:
        """The longest length once n entries more are held, read from the device."""
        return max(0, int((self.lengths.long() + n).max())) if self.batch else 0

    def _note_capture(self) -> bool:
        now = torch.cuda.is_current_stream_capturing()
        self._replayed = self._replayed or now
        return now

    @property
    def bound(self) -> int | None:
        """``longest`` (1 where nothing is held) as the ``max_length`` of
        ``ops.paged_attention``; None, the capacity, in a call that is captured
        and once a change of the lengths was, since replays move them without the
        host's knowledge."""
        return None if self._replayed or torch.cuda.is_current_stream_capturing() else max(1, self.longest)

    def evict(self, budget: int, recent: int = 0, sinks: int = 0, weights=None):
        """``ops.kv_evict`` on all layers; lengths above `budget` become `budget`.
        Give no more than `budget` `recent` and `sinks` together: of more, those
        at the lower places stay, the older ones (``protected`` chooses them).
        Returns the places that the kept entries came from."""
        keep = ops.kv_evict(self, budget, recent=recent, sinks=sinks, weights=weights)
        self.lengths.clamp_(max=budget)
        if not self._note_capture():
            self.longest = min(self.capacity if self._replayed else self.longest, budget)
        return keep

    def is_empty(self) -> bool:
        """Whether no sequence holds an entry; reads the lengths from the device
        unless the host knows that there is none."""
        return (self.longest == 0 and not self._replayed) or self._longest_held() == 0

    def reset(self):
        """Forget all entries (pages keep their contents)."""
        (self.lengths if self._counts is None else self._counts).zero_()
        if not self._note_capture():
            self.longest = 0
