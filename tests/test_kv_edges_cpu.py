"""What the paged key-value cache's calls work out or refuse on the host."""
from __future__ import annotations

import pytest

from test_kv_cpu import append, attend, struct


@pytest.mark.parametrize("budget", [1, 2, 3, 5, 8, 12, 67, 68, 69, 1000])
def test_what_an_eviction_protects_fits_its_budget(budget):
    from bposit_b200.kv import protected
    recent, sinks = protected(budget)
    assert recent >= 1 and sinks >= 0 and recent + sinks <= budget
    if budget >= 68:
        assert (recent, sinks) == (64, 4)
    assert protected(budget, recent=budget) == (budget, 0) and protected(budget, sinks=budget) == (0, budget)
    assert protected(budget, 1, budget - 1) == (1, budget - 1)
    for kw in (dict(recent=budget + 1), dict(sinks=budget + 1), dict(recent=budget, sinks=1), dict(recent=-1),
               dict(sinks=-1), dict(recent=-1, sinks=0)):
        with pytest.raises(ValueError):
            protected(budget, **kw)
    for bad in (0, -budget):
        with pytest.raises(ValueError):
            protected(bad)


# ---- results that would lie on inputs still to be read: found by address, before any device work ----
# (what the check lets through is refused behind it, by the address of a table or of the workspace)
CALLS = [(append, "q_out", dict(cos=20)), (attend, "out", dict(ws=128, n=1 << 30))]


@pytest.mark.parametrize("dtype,es", [(0, 4), (1, 2), (2, 2)])
@pytest.mark.parametrize("call,where,behind", CALLS)
def test_results_may_replace_queries_row_for_row_only(dtype, es, call, where, behind):
    from bposit_b200 import _lib
    L = _lib.lib()
    row, at = 256 * es, 1 << 20                              # two rows of 4 heads of 64
    for qs, out in ((256, 0), (256, 2 * row), (256, -2 * row), (1024, 5 * row), (1024, -2 * row),
                    (1024, row), (1024, 2 * row)):
        rc = call(L, struct(), dtype=dtype, q=at, qs=qs, **{where: at + out}, **behind)
        assert rc == _lib.BP_EALIGN, (qs, out)
    for qs, out in ((512, 0), (264, 0), (256, row), (256, -row), (256, 2 * row - 16), (256, 16 - 2 * row),
                    (1024, row - 16), (1024, 2 * row + 16), (1024, 4 * row), (1024, 5 * row - 16)):
        rc = call(L, struct(), dtype=dtype, q=at, qs=qs, **{where: at + out}, **behind)
        assert rc == _lib.BP_EINVAL and b"row for row" in L.bp_last_error(), (qs, out)


def test_one_row_of_queries_may_have_any_stride():
    from bposit_b200 import _lib
    L = _lib.lib()
    assert attend(L, struct(batch=1), q=4096, qs=512, out=4096, ws=128, n=1 << 30) == _lib.BP_EALIGN
    assert append(L, struct(batch=1), tokens=1, q=4096, qs=512, q_out=4096, cos=20) == _lib.BP_EALIGN


# ---- which device a call asks ----
def test_the_workspace_is_sized_on_the_cache_s_device(monkeypatch):
    """A cache on another device than the current one: the library asks the current device for its SMs, so both calls
    are made with the cache's device current."""
    import types

    import torch

    from bposit_b200 import _lib, ops
    current, asked = [0], []

    class Device:
        index = 1

        def __eq__(self, other):
            return True

        __hash__ = None

    class Guard:
        def __init__(self, device):
            self.to = getattr(device, "index", device)

        def __enter__(self):
            self.was, current[0] = current[0], self.to

        def __exit__(self, *a):
            current[0] = self.was

    def size(*a):
        asked.append(("size", current[0]))
        return 256

    def attend(*a):
        asked.append(("call", current[0]))
        return 0

    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 0, raising=False)
    monkeypatch.setattr(_lib, "lib", lambda: types.SimpleNamespace(bp_paged_attention=attend,
                                                                   bp_paged_attention_workspace_size=size))
    cache = types.SimpleNamespace(device=Device(), head_dim=64, batch=2, capacity=64, layers=1, _workspace={}, _ref=None)
    q = torch.zeros(2, 4, 64)
    for _ in range(2):
        ops.paged_attention(cache, q)
    assert asked == [("size", 1), ("call", 1), ("call", 1)] and current == [0]
