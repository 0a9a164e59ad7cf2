"""window_attention over batches of many prompt chunks at once: CTAs that take
several row blocks in turn, batches that take several launches, and the choice
between the two kernels.  Bounds as in test_bounded_cache_gpu.py."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import bounded_cache as ref  # noqa: E402
from tests.test_bounded_cache_gpu import Cache, close, starts_of  # noqa: E402

pytestmark = pytest.mark.gpu


def batch(seed, seqs, most, longest):
    """Lengths and query lengths: none, one, more queries than tokens, whole
    streams, and chunks of longer ones."""
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, longest, seqs)
    qs = rng.integers(0, most + 1, seqs)
    lens[::17], qs[3::13], qs[5::19] = 0, 0, 1
    lens[7::23] = qs[7::23]
    lens[1], qs[1], lens[-1], qs[-1] = longest, most, longest - 1, most
    return lens.tolist(), qs.tolist()


@pytest.mark.parametrize("dtype,hq,hkv,d,bs,layout,seqs,most", [
    ("bf16", 16, 2, 128, 16, "planes", 300, 40),
    ("fp16", 10, 2, 64, 32, "nhd", 300, 60),
    ("bf16", 8, 1, 64, 8, "planes", 520, 100),
    ("fp16", 4, 4, 128, 8, "planes", 70, 300),
])
def test_many_prompt_chunks(dtype, hq, hkv, d, bs, layout, seqs, most):
    import flashdec_b200 as fd

    window, sinks = 50, 3
    lens, qs = batch(31, seqs, most, 2 * most)
    c = Cache(32, lens, dtype=dtype, hkv=hkv, d=d, bs=bs, layout=layout, fill=float("nan"))
    q, qn = c.queries(sum(qs), hq)
    st = starts_of(qs)
    fd.device_status(clear=True)
    out = fd.window_attention(q, c.k, c.v, c.table, c.seq, window=window, sinks=sinks,
                              query_start_loc=torch.from_numpy(st).cuda(), max_query_len=most)
    exact, size = ref.window_attention_ref(qn, c.k_np, c.v_np, c.table_np, lens, window, sinks, st)
    close(out, *_blank(exact, size, st, lens), dtype, window + sinks)
    assert fd.device_status() == 0
    # fewer queries announced than there are: the same values
    again = fd.window_attention(q, c.k, c.v, c.table, c.seq, window=window, sinks=sinks,
                                query_start_loc=torch.from_numpy(st).cuda(), max_query_len=max(most // 3, 17))
    close(again, *_blank(exact, size, st, lens), dtype, window + sinks)


def _blank(exact, size, st, lens):
    """Rows before their stream's first token are zero."""
    for b, n in enumerate(lens):
        blank = max(0, int(st[b + 1] - st[b]) - int(n))
        assert (exact[st[b]:st[b] + blank] == 0).all()
    return exact, size


@pytest.mark.parametrize("d", [64, 128])
def test_one_bad_sequence_among_many_leaves_the_others_exact(d):
    """A NaN value that only some rows see, and a page outside the cache, in
    the middle of a CTA's items."""
    import flashdec_b200 as fd
    from flashdec_b200 import _lib

    window, sinks, seqs, bs = 60, 2, 330, 16
    lens = [150] * seqs
    qs = [64 if d == 64 else 40] * seqs
    c = Cache(33, lens, hkv=2, d=d, bs=bs)
    q, qn = c.queries(sum(qs), 16)
    st = starts_of(qs)
    token, hurt, paged = 120, (4, 149, 290), 151
    for b in hurt:
        c.v[int(c.table_np[b, token // bs]), 1, token % bs, 9] = float("nan")
    table, bad = c.table.clone(), 140 // bs
    table[paged, bad] = c.pool + 5
    fd.device_status(clear=True)
    out = fd.window_attention(q, c.k, c.v, table, c.seq, window=window, sinks=sinks,
                              query_start_loc=torch.from_numpy(st).cuda(), max_query_len=qs[0])
    assert fd.device_status(clear=True) == _lib.FD_STATUS_BAD_BLOCK_ID
    exact, size = ref.window_attention_ref(qn, c.k_np, c.v_np, c.table_np, lens, window, sinks, st)
    mask = ref.window_mask(150, qs[0], window, sinks)
    far = mask & (np.arange(150) // bs != bad)[None]
    for i in range(16):
        k, v = (ref._dense(x, c.table_np[paged], 150)[:, i // 8] for x in (c.k_np, c.v_np))
        p = ref.softmax_rows(qn[st[paged]:st[paged + 1], i] @ k.T / np.sqrt(d), far)
        exact[st[paged]:st[paged + 1], i], size[st[paged]:st[paged + 1], i] = p @ v, p @ np.abs(v)
    got = out.float().cpu().numpy()
    fine = np.ones(got.shape, bool)
    for b in hurt:
        rows = st[b] + np.flatnonzero(mask[:, token])
        assert np.isnan(got[rows][:, 8:, 9]).all()
        fine[rows[:, None], np.arange(8, 16)[None], 9] = False
    assert np.isfinite(got[fine]).all()
    keep = torch.from_numpy(fine).cuda()
    close(out[keep], exact[fine], size[fine], "bf16", window + sinks)


@pytest.mark.parametrize("d,hq,hkv,seqs,ql", [
    (128, 16, 2, 8, 16), (128, 16, 2, 8, 32), (128, 16, 2, 8, 64), (64, 32, 8, 16, 8), (64, 32, 8, 16, 16),
    (128, 64, 2, 4, 1), (128, 64, 2, 40, 1), (64, 4, 4, 3, 33),
])
def test_both_sides_of_the_choice_of_kernel(d, hq, hkv, seqs, ql):
    import flashdec_b200 as fd

    window, sinks = 500, 4
    lens = [700 + 13 * b for b in range(seqs)]
    c = Cache(34, lens, hkv=hkv, d=d, bs=16)
    q, qn = c.queries(seqs * ql, hq)
    st = starts_of([ql] * seqs)
    out = fd.window_attention(q, c.k, c.v, c.table, c.seq, window=window, sinks=sinks,
                              query_start_loc=torch.from_numpy(st).cuda(), max_query_len=ql)
    exact, size = ref.window_attention_ref(qn, c.k_np, c.v_np, c.table_np, lens, window, sinks, st)
    close(out, exact, size, "bf16", window + sinks)


@pytest.mark.parametrize("ql", [2, 7, 16, 50])
@pytest.mark.parametrize("hq,hkv,d,bs", [(1, 1, 128, 16), (3, 1, 64, 8), (16, 2, 128, 32), (20, 1, 64, 16)])
def test_more_queries_than_announced_over_a_long_window(hq, hkv, d, bs, ql):
    """One query announced, and more there: what the parts of a window send to
    one another has its place for the announced rows only."""
    import flashdec_b200 as fd

    lens, qs = [3000, 40], [ql, ql - 1]
    c = Cache(35, lens, hkv=hkv, d=d, bs=bs)
    q, qn = c.queries(sum(qs), hq)
    st = starts_of(qs)
    for window in (700, 2900):
        out = fd.window_attention(q, c.k, c.v, c.table, c.seq, window=window, sinks=3,
                                  query_start_loc=torch.from_numpy(st).cuda(), max_query_len=1)
        exact, size = ref.window_attention_ref(qn, c.k_np, c.v_np, c.table_np, lens, window, 3, st)
        close(out, exact, size, "bf16", window + 3)


@pytest.mark.parametrize("tokens", [250, 390, 500, 640, 800, 900, 1100])
@pytest.mark.parametrize("hq,hkv,d", [(1, 1, 128), (2, 2, 64), (3, 1, 128), (5, 1, 64)])
def test_any_number_of_parts_and_rows(tokens, hq, hkv, d):
    """One sequence in two to eight parts, with few heads: odd counts of both."""
    import flashdec_b200 as fd

    c = Cache(36, [tokens], hkv=hkv, d=d, bs=16)
    q, qn = c.queries(1, hq)
    out = fd.window_attention(q, c.k, c.v, c.table, c.seq, window=tokens)
    exact, size = ref.window_attention_ref(qn, c.k_np, c.v_np, c.table_np, [tokens], tokens)
    close(out, exact, size, "bf16", tokens)
    scores = torch.ones((c.pool, hkv, 16), device="cuda")
    out = fd.scored_decode(q, c.k, c.v, scores, c.table, c.seq)
    exact, size, want = ref.scored_decode_ref(qn, c.k_np, c.v_np, np.ones((c.pool, hkv, 16)), c.table_np, [tokens])
    close(out, exact, size, "bf16", tokens)
    assert (np.abs(scores.double().cpu().numpy() - want) <= 1e-4 * np.abs(want - 1) + 1e-6).all()
