"""scored_decode's workspace goes by the pages there are, not by the width that
the block tables could be filled to.  Bounds as in test_bounded_cache_gpu.py."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import bounded_cache as ref  # noqa: E402
from tests.test_bounded_cache_gpu import Cache, close  # noqa: E402

pytestmark = pytest.mark.gpu


def widened(table, columns):
    wide = torch.full((table.shape[0], columns), -1, dtype=table.dtype, device=table.device)
    wide[:, :table.shape[1]] = table
    return wide


def scored(c, q, scores, table):
    import flashdec_b200 as fd

    return fd.scored_decode(q, c.k, c.v, scores, table, c.seq)


def check(c, qn, out, scores, start, dtype):
    exact, size, want = ref.scored_decode_ref(qn, c.k_np, c.v_np, start, c.table_np, c.lens)
    close(out, exact, size, dtype, max(c.lens))
    got = scores.double().cpu().numpy()
    assert (np.abs(got - want) <= 1e-4 * np.abs(want - start) + 1e-6 * np.abs(start) + 1e-9).all()


@pytest.mark.parametrize("seqs,hq,hkv,d,bs", [(64, 32, 8, 128, 16), (20, 40, 1, 64, 8), (600, 2, 1, 64, 32)])
def test_short_sequences_under_wide_tables(seqs, hq, hkv, d, bs):
    rng = np.random.default_rng(8)
    c = Cache(44, rng.integers(0, 200, seqs).tolist(), hkv=hkv, d=d, bs=bs)
    q, qn = c.queries(seqs, hq)
    start = rng.random((c.pool, hkv, bs)).astype(np.float32)
    scores = torch.from_numpy(start).cuda()
    table = widened(c.table, 131072 // bs)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = scored(c, q, scores, table)
    torch.cuda.synchronize()
    used = torch.cuda.max_memory_allocated() - before
    # raw scores of at most twice the pool's tokens, partials of two waves of CTAs, the output
    assert used <= 2 * 4 * c.pool * bs * hq + (32 << 20), used
    check(c, qn, out, scores, start.astype(np.float64), "bf16")


@pytest.mark.parametrize("dtype,hq,hkv,d,bs,lens,spare", [
    ("bf16", 8, 2, 128, 16, [5000, 3], 0),        # about as many pages as the tables have places
    ("bf16", 8, 2, 128, 16, [5000, 3], 2000),     # many more
    ("fp16", 40, 1, 64, 8, [2300, 1200, 0], 0),
    ("fp16", 40, 1, 64, 8, [2300, 1200, 0], 3000),
    ("bf16", 16, 4, 64, 32, [9000], 500),
    ("bf16", 66, 2, 128, 8, [1500, 700], 900),
])
@pytest.mark.parametrize("strided", [False, True])
def test_small_and_large_caches(dtype, hq, hkv, d, bs, lens, spare, strided):
    c = Cache(45, lens, dtype=dtype, hkv=hkv, d=d, bs=bs, extra_pages=spare)
    q, qn = c.queries(len(lens), hq)
    start = c.rng.random((c.pool, hkv, bs)).astype(np.float32)
    scores = torch.empty((c.pool, hkv, bs + 1 if strided else bs), device="cuda")[..., :bs]
    scores.copy_(torch.from_numpy(start))
    check(c, qn, scored(c, q, scores, c.table), scores, start.astype(np.float64), dtype)


@pytest.mark.parametrize("spare", [0, 2000])
def test_pages_outside_the_cache_get_no_scores(spare):
    """A page that is not in the cache holds no key, and the scores of all
    others are those of the rest."""
    import flashdec_b200 as fd
    from flashdec_b200 import _lib

    n, bs = 3001, 8
    c = Cache(46, [n, 40], hkv=1, d=64, bs=bs, extra_pages=spare)
    q, qn = c.queries(2, 4)
    gone = [0, 1, 100, 255, n // bs]
    table = c.table.clone()
    table[0, gone] = torch.tensor([-1, c.pool, 1 << 20, -7, c.pool], dtype=table.dtype, device="cuda")
    start = c.rng.random((c.pool, 1, bs)).astype(np.float32)
    scores = torch.from_numpy(start).cuda()
    fd.device_status(clear=True)
    out = scored(c, q, scores, table)
    assert fd.device_status(clear=True) == _lib.FD_STATUS_BAD_BLOCK_ID
    k, v = (ref._dense(x, c.table_np[0], n)[:, 0] for x in (c.k_np, c.v_np))
    mask = ~np.isin(np.arange(n) // bs, gone)[None]
    want, weight = start.astype(np.float64), np.zeros(n)
    for i in range(4):
        p = ref.softmax_rows(qn[:1, i] @ k.T / 8.0, mask)
        close(out[:1, i], p @ v, p @ np.abs(v), "bf16", n)
        weight += p[0]
    for t in np.flatnonzero(mask[0]):
        want[c.table_np[0, t // bs], 0, t % bs] += weight[t]
    exact, size, other = ref.scored_decode_ref(qn[1:], c.k_np, c.v_np, start, c.table_np[1:], [40])
    close(out[1:], exact, size, "bf16", 40)
    for page in c.table_np[1, :5]:
        want[page] = other[page]
    got = scores.double().cpu().numpy()
    assert (np.abs(got - want) <= 1e-4 * np.abs(want - start) + 1e-6 * np.abs(start) + 1e-9).all()


def test_sequences_that_list_more_pages_than_there_are():
    """Lengths far past the cache under wide tables: outputs as ever, the bad
    pages reported, nothing written elsewhere."""
    import flashdec_b200 as fd
    from flashdec_b200 import _lib

    lens = [100, 60, 90]
    c = Cache(47, lens, hkv=1, d=64, bs=16)
    q, qn = c.queries(3, 4)
    table = widened(c.table, 4096)
    c.seq[1] = 65536
    scores = torch.zeros((c.pool + 8, 1, 16), device="cuda")[4:-4]
    guard = scores._base
    fd.device_status(clear=True)
    out = scored(c, q, scores, table)
    assert fd.device_status(clear=True) == _lib.FD_STATUS_BAD_BLOCK_ID
    exact, size = ref.window_attention_ref(qn, c.k_np, c.v_np, c.table_np, lens, 1 << 30)
    for b in (0, 2):
        close(out[b:b + 1], exact[b:b + 1], size[b:b + 1], "bf16", 100)
    pages = c.table_np[0, :7]
    want = ref.scored_decode_ref(qn[:1], c.k_np, c.v_np, np.zeros((c.pool, 1, 16)), c.table_np[:1], [100])[2]
    got = scores.double().cpu().numpy()
    assert (np.abs(got[pages] - want[pages]) <= 1e-4 * want[pages] + 1e-9).all()
    assert (guard[:4] == 0).all() and (guard[-4:] == 0).all()
