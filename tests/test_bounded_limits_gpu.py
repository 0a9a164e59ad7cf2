"""The bounded-cache operators at the ends of what their checks accept."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import bounded_cache as ref  # noqa: E402
from tests.test_bounded_cache_gpu import Cache  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("budget", [2 ** 31 - 1, 2 ** 31 - 513])
def test_evict_with_the_greatest_budget(budget):
    """`kept` is filled up to the budget, in steps that pass INT_MAX."""
    import flashdec_b200 as fd

    c = Cache(40, [21], hkv=1, d=64, bs=8, extra_pages=3)
    scores = torch.rand((c.pool, 1, 8), device="cuda")
    new = torch.from_numpy(c.spare[:3]).cuda()[None]
    k, v, s = c.k.clone(), c.v.clone(), scores.clone()
    kept, left = fd.evict_tokens(c.k, c.v, scores, c.table, c.seq, new, budget=budget, sinks=2, recent=5)
    assert left.tolist() == [21]
    assert kept.shape == (1, 1, budget) and kept[0, 0, :21].tolist() == list(range(21))
    assert int(kept[0, 0, 21:].max()) == -1 and int(kept[0, 0, 21:].min()) == -1
    del kept
    torch.cuda.empty_cache()
    for got, was in ((c.k, k), (c.v, v), (scores, s)):
        want = was.clone()
        for t in range(21):
            want[int(new[0, t // 8]), 0, t % 8] = was[int(c.table[0, t // 8]), 0, t % 8]
        assert torch.equal(got, want)
