"""The bounded-cache operators at the ends of what their checks accept."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import bounded_cache as ref  # noqa: E402
from tests.test_bounded_cache_gpu import Cache, close  # noqa: E402

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


@pytest.mark.parametrize("group", [12500, 16384])
def test_scored_decode_with_the_greatest_groups(group):
    """The scores' pass keeps a sum per query head of the group."""
    import flashdec_b200 as fd

    c = Cache(41, [37], hkv=1, d=64, bs=16)
    q, qn = c.queries(1, group)
    scores = torch.zeros((c.pool, 1, 16), device="cuda")
    out = fd.scored_decode(q, c.k, c.v, scores, c.table, c.seq)
    exact, size, want = ref.scored_decode_ref(qn, c.k_np, c.v_np, np.zeros(scores.shape), c.table_np, [37])
    close(out, exact, size, "bf16", 37)
    assert (np.abs(scores.double().cpu().numpy() - want) <= 1e-4 * want).all()


def test_scored_decode_refuses_a_greater_group():
    import flashdec_b200 as fd
    from flashdec_b200 import _lib

    c = Cache(41, [37], hkv=1, d=64, bs=16)
    q, _ = c.queries(1, 16385)
    with pytest.raises(_lib.FlashDecNativeError):
        fd.scored_decode(q, c.k, c.v, torch.zeros((c.pool, 1, 16), device="cuda"), c.table, c.seq)
