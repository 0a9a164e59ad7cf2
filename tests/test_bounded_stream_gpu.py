"""The bounded-cache operators together (examples/bounded_stream.py): streams
that outgrow their cache, against a plain model of the same stream."""

from __future__ import annotations

import sys
from pathlib import Path

import numpy as np
import pytest

torch = pytest.importorskip("torch")

ROOT = Path(__file__).resolve().parents[1]

pytestmark = pytest.mark.gpu


def _example():
    if str(ROOT / "examples") not in sys.path:
        sys.path.insert(0, str(ROOT / "examples"))
    import bounded_stream

    return bounded_stream


def test_streams_stay_within_their_budget():
    import flashdec_b200 as fd

    fd.device_status(clear=True)
    layer, out = _example().run(streams=3, prompt=700, tokens=150, budget=256, slack=64, recent=64)
    assert torch.isfinite(out.float()).all()
    assert layer.position == [850] * 3
    assert all(256 <= n <= 320 for n in layer.length)
    assert layer.evicted == sum(p - n for p, n in zip(layer.position, layer.length))
    used = sum(len(p) for p in layer.pages)
    assert sorted(layer.free + [x for p in layer.pages for x in p]) == list(range(layer.blocks))
    assert used <= 3 * layer.row
    # what is cached now: every token's score is a sum of weights
    assert (layer.scores >= 0).all() and torch.isfinite(layer.scores).all()
    assert fd.device_status() == 0


def test_decode_after_eviction_attends_to_the_kept_tokens():
    """One stream, decoded past its budget: the output of each step equals
    attention over the tokens that the example still holds."""
    ex = _example()
    gen = torch.Generator(device="cuda").manual_seed(3)
    layer = ex.BoundedLayer(1, q_heads=8, kv_heads=2, head_dim=64, block_size=8, budget=40, slack=8, sinks=2,
                            recent=10)
    shadow = [[] for _ in range(2)]  # per KV head: (k, v) rows in the cache, as numpy
    for step in range(120):
        q, k, v = (torch.randn((1, h, 64), generator=gen, device="cuda").bfloat16() for h in (8, 2, 2))
        full = layer.length[0] >= 48
        if full:  # follow the eviction by what it kept
            before = layer._table([0])
            lens = torch.tensor([48], dtype=torch.int32, device="cuda")
            scores = torch.zeros((2, 48))
            for t in range(48):
                scores[:, t] = layer.scores[int(before[0, t // 8]), :, t % 8].cpu()
            from oracle.bounded_cache import evict_choice

            for h in range(2):
                take = evict_choice(scores[h].tolist(), 40, 2, 10)
                shadow[h] = [shadow[h][t] for t in take]
            assert int(lens[0]) == layer.length[0]
        out = layer.decode([0], q, k, v)
        n = layer.length[0]
        page, off = layer.pages[0][(n - 1) // 8], (n - 1) % 8
        for h in range(2):
            shadow[h].append((layer.k[page, h, off].double().cpu().numpy(), layer.v[page, h, off].double().cpu().numpy()))
            assert len(shadow[h]) == n
        # q as the kernel saw it
        import flashdec_b200 as fd

        pos = torch.tensor([layer.position[0] - 1], device="cuda")
        rot = fd.apply_rope(q, pos, rotary_dim=64, base=1e6).double().cpu().numpy()[0]
        for i in range(8):
            ks, vs = (np.stack([r[j] for r in shadow[i // 4]]) for j in (0, 1))
            x = ks @ rot[i] / 8.0
            w = np.exp(x - x.max())
            w /= w.sum()
            bound = (2 * 2.0 ** -8 + 1e-4) * (w @ np.abs(vs)) + 1e-6
            assert (np.abs(out[0, i].double().cpu().numpy() - w @ vs) <= bound).all(), step
