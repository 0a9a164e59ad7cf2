"""The launch forms that long sequences and large batches take: clusters and
re-read scores in the eviction, copies of many batches a warp, shares of the
batch's tiles with several KV heads, scales of every sign, caches past 32-bit
offsets, graphs and side streams.  Bounds as in test_bounded_cache_gpu.py;
evictions are exact."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import bounded_cache as ref  # noqa: E402
from tests.test_bounded_cache_gpu import Cache, close, starts_of  # noqa: E402

pytestmark = pytest.mark.gpu


def choice(w, budget, sinks, recent):
    """evict_choice of the oracle for long rows."""
    n = len(w)
    if n <= budget:
        return np.arange(n)
    mid = np.arange(sinks, n - recent)
    x = w[mid].astype(np.float64)
    order = np.lexsort((mid, np.where(np.isnan(x), 0.0, -x) + 0.0, ~np.isnan(x)))
    best = mid[order[:budget - sinks - recent]]
    return np.sort(np.concatenate([np.arange(sinks), best, np.arange(n - recent, n)]))


def test_the_choice_for_long_rows_is_the_oracle_s():
    rng = np.random.default_rng(3)
    for values in ("ties", "special"):
        for n, budget, sinks, recent in ((40, 20, 3, 5), (40, 1, 0, 0), (50, 49, 0, 40), (9, 12, 1, 2)):
            w = scores_of(rng, (n,), values)
            assert choice(w, budget, sinks, recent).tolist() == ref.evict_choice(w, budget, sinks, recent)


def scores_of(rng, shape, values):
    w = np.exp(2 * rng.standard_normal(shape)).astype(np.float32)
    if values == "equal":
        w[:] = 0.25
    elif values == "ties":
        w = np.round(w)
    elif values == "near":  # one exponent and a few of its next bits: most keys share two digits
        w = (1 + rng.integers(0, 1 << 12, shape) * 2.0 ** -23).astype(np.float32)
    elif values == "special":
        pick = rng.integers(0, 9, shape)
        for i, x in enumerate((0.0, -0.0, np.nan, np.inf, -np.inf, -1.5, 1e-42)):
            w[pick == i] = x
    return w


def evicted(lens, *, hkv, d, bs, budget, sinks, recent, values, columns=None, strided=False, seed=0):
    """Evict random pages of the lengths under tables of `columns` entries and
    compare everything."""
    import flashdec_b200 as fd

    rng = np.random.default_rng(seed)
    counts = [-(-n // bs) for n in lens]
    new = [-(-min(n, budget) // bs) for n in lens]
    pool = sum(counts) + sum(new) + 2
    perm = rng.permutation(pool)
    columns = columns or max(max(counts), 1)
    table = np.full((len(lens), columns), -1, np.int32)
    to = np.full((len(lens), max(max(new), -(-min(budget, columns * bs) // bs), 1)), -1, np.int32)
    at = 0
    for b in range(len(lens)):
        table[b, :counts[b]] = perm[at:at + counts[b]]
        at += counts[b]
        to[b, :new[b]] = perm[at:at + new[b]]
        at += new[b]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    k, v = (torch.randn((pool, hkv, bs, d), generator=gen, device="cuda").bfloat16() for _ in range(2))
    w = scores_of(rng, (pool, hkv, bs), values)
    scores = torch.empty((pool, hkv, bs, 2 if strided else 1), device="cuda")[..., 0]
    scores.copy_(torch.from_numpy(w))
    want = [x.clone() for x in (k, v, scores)]
    fd.device_status(clear=True)
    kept, left = fd.evict_tokens(k, v, scores, torch.from_numpy(table).cuda(), torch.tensor(lens, device="cuda"),
                                 torch.from_numpy(to).cuda(), budget=budget, sinks=sinks, recent=recent)
    assert left.tolist() == [min(n, budget) for n in lens]
    got = kept.cpu().numpy()
    for b, n in enumerate(lens):
        t = np.arange(n)
        m = min(n, budget)
        for h in range(hkv):
            take = choice(w[table[b, t // bs], h, t % bs], budget, sinks, recent)
            assert np.array_equal(got[b, h, :m], take), (b, h)
            assert (got[b, h, m:] == -1).all()
            i = np.arange(m)
            src = torch.from_numpy(table[b, take // bs].astype(np.int64)).cuda(), torch.from_numpy(take % bs).cuda()
            dst = torch.from_numpy(to[b, i // bs].astype(np.int64)).cuda(), torch.from_numpy(i % bs).cuda()
            for x in want:  # source pages are never new ones
                x[dst[0], h, dst[1]] = x[src[0], h, src[1]]
    for x, y in zip((k, v, scores), want):
        assert torch.equal(torch.nan_to_num(x, 7.5), torch.nan_to_num(y, 7.5))
        assert torch.equal(torch.isnan(x), torch.isnan(y))
    assert fd.device_status() == 0


@pytest.mark.parametrize("values", ["random", "ties", "equal", "near", "special"])
@pytest.mark.parametrize("lens,budget,sinks,recent", [
    ([4100, 4095, 17, 0], 1000, 4, 300),      # two CTAs a row
    ([9000, 2500, 9001], 4001, 0, 1),         # four
    ([33001, 5, 20000], 2999, 7, 0),          # eight
    ([33001], 32990, 1, 2),                   # nearly all kept
])
def test_evict_long_rows(lens, budget, sinks, recent, values):
    evicted(lens, hkv=1, d=64, bs=16, budget=budget, sinks=sinks, recent=recent, values=values, seed=len(lens))


@pytest.mark.parametrize("values", ["random", "near", "special"])
def test_evict_rows_past_what_a_cluster_keeps(values):
    """Above 393216 places in the table the scores are read again for each digit."""
    evicted([400001], hkv=1, d=64, bs=32, budget=70001, sinks=5, recent=1001, values=values)
    evicted([300, 5000, 70000], hkv=2, d=64, bs=8, budget=299, sinks=5, recent=99, values=values, columns=50000)


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("columns", [300, 2000, 20000])
def test_evict_short_rows_under_wide_tables(columns, strided):
    evicted([1, 33, 260, 700, 0], hkv=3, d=128, bs=8, budget=131, sinks=2, recent=50, values="ties", columns=columns,
            strided=strided)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("values", ["ties", "special"])
def test_evict_batches_whose_warps_copy_many_rows(d, values):
    rng = np.random.default_rng(9)
    lens = rng.integers(150, 420, 230).tolist()
    evicted(lens, hkv=16, d=d, bs=16, budget=201, sinks=3, recent=60, values=values, strided=values == "special")


SHARES = [
    # dtype, hq, hkv, d, bs, layout, lens
    ("bf16", 32, 8, 128, 16, "planes", [40000, 17, 3000]),
    ("fp16", 16, 2, 128, 32, "nhd", [70001]),
    ("bf16", 40, 2, 128, 16, "planes", [30000, 1, 0, 9000]),
    ("bf16", 8, 8, 64, 8, "nhd", [20000, 1500] * 5),
    ("fp16", 12, 4, 128, 8, "planes", [700, 0, 3, 2500] * 20),
]


@pytest.mark.parametrize("case", SHARES, ids=[f"h{i}" for i in range(len(SHARES))])
def test_shares_of_the_batch_with_several_kv_heads(case):
    import flashdec_b200 as fd

    dtype, hq, hkv, d, bs, layout, lens = case
    c = Cache(60, lens, dtype=dtype, hkv=hkv, d=d, bs=bs, layout=layout)
    q, qn = c.queries(len(lens), hq)
    start = c.rng.random((c.pool, hkv, bs)).astype(np.float32)
    scores = torch.from_numpy(start).cuda()
    fd.device_status(clear=True)
    out = fd.scored_decode(q, c.k, c.v, scores, c.table, c.seq)
    exact, size, want = ref.scored_decode_ref(qn, c.k_np, c.v_np, start, c.table_np, lens)
    close(out, exact, size, dtype, max(lens))
    got = scores.double().cpu().numpy()
    assert (np.abs(got - want) <= 1e-4 * np.abs(want - start) + 1e-6 * start + 1e-9).all()
    window = max(lens) * 2 // 3
    out = fd.window_attention(q, c.k, c.v, c.table, c.seq, window=window, sinks=9)
    exact, size = ref.window_attention_ref(qn, c.k_np, c.v_np, c.table_np, lens, window, 9)
    close(out, exact, size, dtype, window + 9)
    assert fd.device_status() == 0


@pytest.mark.parametrize("scale", [-0.3, 0.0, -1e-6, 0.7])
@pytest.mark.parametrize("hq,hkv,d,lens,qs", [
    (8, 2, 128, [300, 40], [1, 1]), (8, 2, 64, [3000, 40], [5, 2]), (16, 2, 128, [700, 260], [300, 129]),
    (4, 4, 64, [500, 20], [500, 20]),
])
def test_scales_of_every_sign(scale, hq, hkv, d, lens, qs):
    import flashdec_b200 as fd

    c = Cache(61, lens, hkv=hkv, d=d, bs=16, fill=float("nan"))
    q, qn = c.queries(sum(qs), hq, 0.7)
    st = starts_of(qs)
    strided = torch.empty((sum(qs), hq, 2, d), dtype=q.dtype, device="cuda")[:, :, 1].transpose(0, 1).contiguous()
    strided = strided.transpose(0, 1)  # heads outermost
    out = fd.window_attention(q, c.k, c.v, c.table, c.seq, window=200, sinks=3, sm_scale=scale, out=strided,
                              query_start_loc=torch.from_numpy(st).cuda(), max_query_len=max(qs))
    exact, size = ref.window_attention_ref(qn, c.k_np, c.v_np, c.table_np, lens, 200, 3, st, sm_scale=scale)
    close(out, exact, size, "bf16", 203)
    if qs == [1, 1]:
        for rows in (lens, [9000, 5000]):
            c = Cache(61, rows, hkv=hkv, d=d, bs=16)
            scores = torch.zeros((c.pool, hkv, 16), device="cuda")
            out = fd.scored_decode(q, c.k, c.v, scores, c.table, c.seq, sm_scale=scale)
            exact, size, want = ref.scored_decode_ref(qn, c.k_np, c.v_np, np.zeros(scores.shape), c.table_np, rows,
                                                      sm_scale=scale)
            close(out, exact, size, "bf16", max(rows))
            assert (np.abs(scores.double().cpu().numpy() - want) <= 1e-4 * want + 1e-9).all()


@pytest.mark.parametrize("d", [64, 128])
def test_prompts_with_unaligned_queries_and_outputs(d):
    import flashdec_b200 as fd

    lens, qs = [500, 333], [400, 201]
    c = Cache(62, lens, hkv=2, d=d, bs=16)
    q, qn = c.queries(sum(qs), 16)
    st = starts_of(qs)
    qv = torch.empty((sum(qs), 16, d + 1), dtype=q.dtype, device="cuda")[..., 1:]
    qv.copy_(q)
    wide = torch.full((sum(qs), 16, 2 * d + 1), 3.0, dtype=q.dtype, device="cuda")
    out = wide[..., 1::2]
    fd.window_attention(qv, c.k, c.v, c.table, c.seq, window=150, sinks=5, out=out, max_query_len=max(qs),
                        query_start_loc=torch.from_numpy(st).cuda())
    exact, size = ref.window_attention_ref(qn, c.k_np, c.v_np, c.table_np, lens, 150, 5, st)
    close(out, exact, size, "bf16", 155)
    assert (wide[..., ::2] == 3).all()


def test_pages_past_32_bit_offsets():
    """Caches of more than 2^32 elements, the sequences' pages at their end."""
    import flashdec_b200 as fd

    hkv, bs, d, hq = 8, 16, 128, 16
    blocks = (1 << 32) // (hkv * bs * d) + 400
    lens = [1500, 900]
    small = Cache(63, lens, hkv=hkv, d=d, bs=bs, extra_pages=100)
    k, v = (torch.empty((blocks, hkv, bs, d), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    scores = torch.zeros((blocks, hkv, bs), device="cuda")
    first = blocks - small.pool
    k[first:], v[first:] = small.k, small.v
    table = torch.where(small.table >= 0, small.table + first, small.table)
    for qs in ([1, 1], [300, 200]):
        q, qn = small.queries(sum(qs), hq)
        st = starts_of(qs)
        out = fd.window_attention(q, k, v, table, small.seq, window=700, sinks=4, max_query_len=max(qs),
                                  query_start_loc=torch.from_numpy(st).cuda())
        exact, size = ref.window_attention_ref(qn, small.k_np, small.v_np, small.table_np, lens, 700, 4, st)
        close(out, exact, size, "bf16", 704)
    q, qn = small.queries(2, hq)
    out = fd.scored_decode(q, k, v, scores, table, small.seq)
    exact, size, want = ref.scored_decode_ref(qn, small.k_np, small.v_np, np.zeros((small.pool, hkv, bs)),
                                              small.table_np, lens)
    close(out, exact, size, "bf16", 1500)
    got = scores[first:].double().cpu().numpy()
    assert (np.abs(got - want) <= 1e-4 * want + 1e-9).all()
    new = torch.from_numpy(small.spare[:80].reshape(2, 40).astype(np.int32)).cuda() + first
    w = scores[first:].cpu().numpy()
    kept, _ = fd.evict_tokens(k, v, scores, table, small.seq, new, budget=640, sinks=4, recent=100)
    for b, n in enumerate(lens):
        t = np.arange(n)
        for h in range(hkv):
            take = choice(w[small.table_np[b, t // bs], h, t % bs], 640, 4, 100)
            assert np.array_equal(kept[b, h].cpu().numpy(), take)
            i = torch.arange(640, device="cuda")
            dst = new[b].long()[i // bs]
            src = table[b].long()[torch.from_numpy(take // bs).cuda()]
            off = torch.from_numpy(take % bs).cuda()
            for x in (k, v, scores):
                assert torch.equal(x[dst, h, i % bs], x[src, h, off])


def test_graphs_of_the_operators_together():
    """A decode step with scores, an eviction and a prompt chunk captured once and
    replayed with other lengths and scores."""
    import flashdec_b200 as fd

    lens, bs, hkv, d = [5000, 700], 16, 2, 128
    c = Cache(64, lens, hkv=hkv, d=d, bs=bs, extra_pages=80)
    q, qn = c.queries(2, 8)
    chunk, chunk_np = c.queries(300, 8)
    st = torch.tensor([0, 200, 300], device="cuda")
    scores = torch.zeros((c.pool, hkv, bs), device="cuda")
    new = torch.from_numpy(c.spare[:80].reshape(2, 40).astype(np.int32)).cuda()
    k, v = c.k.clone(), c.v.clone()

    def step():
        a = fd.scored_decode(q, c.k, c.v, scores, c.table, c.seq)
        kept, left = fd.evict_tokens(c.k, c.v, scores, c.table, c.seq, new, budget=600, sinks=2, recent=50)
        b = fd.window_attention(chunk, c.k, c.v, c.table, c.seq, window=250, sinks=2, query_start_loc=st,
                                max_query_len=200)
        return a, kept, left, b

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for lens in ([5000, 700], [4999, 1], [601, 650], [300, 400]):
        c.seq.copy_(torch.tensor(lens))
        c.k.copy_(k)
        c.v.copy_(v)
        start = c.rng.random(tuple(scores.shape)).astype(np.float32)
        scores.copy_(torch.from_numpy(start))
        graph.replay()
        exact, size, want = ref.scored_decode_ref(qn, c.k_np, c.v_np, start, c.table_np, lens)
        close(out[0], exact, size, "bf16", max(lens))
        got = scores.double().cpu().numpy()
        old = np.unique(c.table_np[c.table_np >= 0])
        assert (np.abs(got - want)[old] <= 1e-4 * np.abs(want - start)[old] + 1e-6).all()
        w = got.astype(np.float32)
        for b, n in enumerate(lens):
            t = np.arange(n)
            for h in range(hkv):
                take = choice(w[c.table_np[b, t // bs], h, t % bs], 600, 2, 50)
                assert np.array_equal(out[1][b, h, :len(take)].cpu().numpy(), take)
        assert out[2].tolist() == [min(n, 600) for n in lens]
        exact, size = ref.window_attention_ref(chunk_np, c.k_np, c.v_np, c.table_np, lens, 250, 2, [0, 200, 300])
        close(out[3], exact, size, "bf16", 252)
