"""examples/bounded_stream.py where pages change hands: a prompt that gets the
pages of evicted tokens starts without their scores, and a prompt longer than
its cache keeps what its own window attention sees."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests.test_bounded_stream_gpu import _example  # noqa: E402

pytestmark = pytest.mark.gpu


def _drawn(gen, n, layer):
    return tuple(torch.randn((n, h, layer.head_dim), generator=gen, device="cuda").to(layer.k.dtype)
                 for h in (layer.q_heads, layer.kv_heads, layer.kv_heads))


def _slots(layer, stream):
    t = np.arange(layer.length[stream])
    return [layer.pages[stream][x] for x in t // layer.block_size], (t % layer.block_size).tolist()


@pytest.mark.parametrize("poison", [None, float("nan")])
def test_a_prompt_on_recycled_pages_has_no_scores_yet(poison):
    layer = _example().BoundedLayer(2, q_heads=8, kv_heads=2, head_dim=64, block_size=8, budget=64, slack=16, sinks=2,
                                    recent=16)
    gen = torch.Generator(device="cuda").manual_seed(5)
    layer.prompt(0, *_drawn(gen, 60, layer))
    for _ in range(40):
        layer.decode([0], *_drawn(gen, 1, layer))
    assert layer.evicted > 0
    if poison is not None:  # as a stream with a broken layer would leave them
        layer.scores[layer.free] = poison
    layer.prompt(1, *_drawn(gen, 70, layer))
    blocks, offsets = _slots(layer, 1)
    assert (layer.scores[blocks, :, offsets] == 0).all()
    layer.decode([1], *_drawn(gen, 1, layer))
    blocks, offsets = _slots(layer, 1)
    # one step's weights of the 4 query heads of each KV head
    total = layer.scores[blocks, :, offsets].double().sum(0)
    assert torch.allclose(total, torch.full_like(total, 4.0), rtol=1e-4, atol=0)


@pytest.mark.parametrize("tokens", [80, 81, 250, 320])
def test_a_prompt_longer_than_its_cache_keeps_the_newest(tokens):
    layer = _example().BoundedLayer(1, q_heads=8, kv_heads=2, head_dim=64, block_size=8, budget=64, slack=16, sinks=2,
                                    recent=16)
    gen = torch.Generator(device="cuda").manual_seed(6)
    q, k, v = _drawn(gen, tokens, layer)
    layer.prompt(0, q, k, v, chunk=50)
    for _ in range(2):  # the first decoded tokens of a full stream have little to rank by
        blocks, offsets = _slots(layer, 0)
        n = layer.length[0]
        assert torch.equal(layer.v[blocks, :, offsets], torch.cat([v[:2], v[len(v) - (n - 2):]]))
        step = _drawn(gen, 1, layer)
        v = torch.cat([v, step[2]])
        layer.decode([0], *step)
