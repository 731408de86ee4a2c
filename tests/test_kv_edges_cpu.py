"""What the paged key-value cache's calls work out or refuse on the host."""
from __future__ import annotations

import pytest


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
