"""window_attention, scored_decode and evict_tokens against their 64-bit
statements (oracle/bounded_cache.py).

Bounds, fixed before the first run.  The softmax weights and the output are
each rounded once to the cache's type (relative error u = 2^-8 for bf16, 2^-11
for fp16), everything else is fp32: |out - exact| <= (2 u + 1e-4) sum p |v|,
plus for fp16 weights below the normal range an absolute 2^-25 max |v| per
token.  1e-4 covers the fp32 scores (products of up to 128 terms, |score| <= 40)
and exponentials.  Accumulated scores are fp32 throughout: 1e-4 relative to
the weight added and 1e-6 to the sum."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import bounded_cache as ref  # noqa: E402

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
U = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}


class Cache:
    """A scattered paged cache on the device and its numpy copy."""

    def __init__(self, seed, lens, *, dtype="bf16", hkv=2, d=128, bs=16, layout="planes", index=torch.int32,
                 extra_pages=0, fill=None):
        rng = np.random.default_rng(seed)
        counts = [max(1, -(-n // bs)) for n in lens]
        self.bs, self.dtype, self.lens = bs, dtype, list(lens)
        pool = sum(counts) + 3 + extra_pages
        perm = rng.permutation(pool)
        self.spare = perm[sum(counts):]
        table = np.full((len(lens), max(counts)), -1, np.int64)
        at = 0
        for b, c in enumerate(counts):
            table[b, :c] = perm[at:at + c]
            at += c
        self.table_np = table
        host = {x: torch.from_numpy(rng.standard_normal((pool, hkv, bs, d), np.float32)).to(DT[dtype])
                for x in "kv"}
        if fill is not None:  # everything that is not a token of a sequence
            live = torch.zeros((pool, bs), dtype=torch.bool)
            for b, n in enumerate(lens):
                for t in range(n):
                    live[table[b, t // bs], t % bs] = True
            for x in "kv":
                host[x][~live[:, None].expand(-1, hkv, -1)] = fill
        self.k_np, self.v_np = (host[x].double().numpy() for x in "kv")
        self.k, self.v = self.place(host["k"], host["v"], layout)
        self.table = torch.from_numpy(table).to(index).cuda()
        self.seq = torch.tensor(self.lens, dtype=index, device="cuda")
        self.rng, self.pool, self.hkv, self.d = rng, pool, hkv, d

    def place(self, k, v, layout):
        nb, h, bs, d = k.shape
        if layout == "nhd":
            kv = torch.empty((nb, 2, bs, h, d), dtype=k.dtype, device="cuda")
            kv[:, 0] = k.permute(0, 2, 1, 3).cuda()
            kv[:, 1] = v.permute(0, 2, 1, 3).cuda()
            return kv[:, 0].permute(0, 2, 1, 3), kv[:, 1].permute(0, 2, 1, 3)
        if layout == "dims":  # dim-major storage: no unit stride along a row
            return tuple(x.permute(0, 1, 3, 2).contiguous().cuda().permute(0, 1, 3, 2) for x in (k, v))
        if layout == "odd":  # rows that start off a 16-byte boundary
            out = []
            for x in (k, v):
                buf = torch.zeros((nb, h, bs, d + 3), dtype=x.dtype, device="cuda")
                buf[..., 1:d + 1] = x.cuda()
                out.append(buf[..., 1:d + 1])
            return tuple(out)
        return k.cuda(), v.cuda()

    def queries(self, tokens, hq, scale=1.0):
        q = torch.from_numpy(self.rng.standard_normal((tokens, hq, self.d), np.float32) * scale)
        q = q.to(DT[self.dtype])
        return q.cuda(), q.double().numpy()


def close(out, exact, size, dtype, tokens, vmax=6.0):
    got = out.double().cpu().numpy()
    bound = (2 * U[dtype] + 1e-4) * size + 1e-6
    if dtype == "fp16":
        bound = bound + tokens * 2.0 ** -25 * vmax
    bad = ~(np.abs(got - exact) <= bound)
    assert not bad.any(), (int(bad.sum()), float(np.nanmax(np.abs(got - exact) / bound)))


def starts_of(qs):
    return np.concatenate([[0], np.cumsum(qs)])


WINDOW = [
    # dtype, hq, hkv, d, bs, layout, lens, query lengths (None: one each), window, sinks
    ("bf16", 16, 2, 128, 32, "planes", [1, 2, 31, 32, 33, 257], None, 64, 4),
    ("fp16", 16, 2, 128, 16, "nhd", [5, 100, 700], None, 1, 0),
    ("bf16", 8, 8, 64, 8, "planes", [1, 7, 8, 9, 200], None, 33, 1),
    ("fp16", 7, 1, 128, 8, "dims", [90, 3], None, 17, 16),
    ("bf16", 10, 2, 64, 16, "odd", [90, 300], None, 100, 37),
    ("bf16", 40, 2, 128, 32, "planes", [300, 64], None, 129, 2),
    ("bf16", 16, 2, 128, 32, "planes", [40, 300, 129], [1, 5, 8], 50, 4),
    ("fp16", 32, 8, 128, 16, "nhd", [300, 17, 64], [7, 0, 3], 64, 1),
    ("bf16", 4, 4, 64, 8, "planes", [300, 1], [33, 1], 16, 0),
    ("fp16", 16, 2, 128, 32, "planes", [523, 70, 200], [130, 70, 33], 100, 8),
    ("bf16", 32, 8, 128, 16, "planes", [400], [400], 128, 4),
    ("bf16", 6, 2, 64, 16, "nhd", [259, 300], [259, 129], 1000, 0),
    ("fp16", 5, 1, 128, 8, "planes", [600], [515], 77, 20),
    ("bf16", 2, 2, 128, 32, "odd", [200], [150], 64, 4),
    ("bf16", 8, 8, 128, 16, "planes", [900, 260], [513, 260], 300, 1),
]


@pytest.mark.parametrize("case", WINDOW, ids=[f"w{i}" for i in range(len(WINDOW))])
@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=["i32", "i64"])
def test_window_attention(case, index):
    import flashdec_b200 as fd

    dtype, hq, hkv, d, bs, layout, lens, qs, window, sinks = case
    c = Cache(7, lens, dtype=dtype, hkv=hkv, d=d, bs=bs, layout=layout, index=index, fill=float("nan"))
    ql = qs or [1] * len(lens)
    q, qn = c.queries(sum(ql), hq)
    st = starts_of(ql)
    fd.device_status(clear=True)
    out = fd.window_attention(q, c.k, c.v, c.table, c.seq, window=window, sinks=sinks,
                              query_start_loc=None if qs is None else torch.from_numpy(st).to(index).cuda(),
                              max_query_len=None if qs is None else max(qs))
    exact, size = ref.window_attention_ref(qn, c.k_np, c.v_np, c.table_np, lens, window, sinks, st)
    close(out, exact, size, dtype, min(max(lens), window + sinks))
    assert fd.device_status() == 0


def test_window_pages_outside_the_window_are_not_read():
    import flashdec_b200 as fd

    lens, window, sinks, bs = [700, 333], 65, 5, 16
    for qs in ([1, 1], [4, 6], [130, 200]):
        c = Cache(3, lens, bs=bs)
        q, qn = c.queries(sum(qs), 8)
        st = starts_of(qs)
        exact, size = ref.window_attention_ref(qn, c.k_np, c.v_np, c.table_np, lens, window, sinks, st)
        table = c.table.clone()
        for b, n in enumerate(lens):
            lo = max(0, n - qs[b] - window + 1)
            table[b, 1:lo // bs] = -7 if b else 1 << 30
        fd.device_status(clear=True)
        out = fd.window_attention(q, c.k, c.v, table, c.seq, window=window, sinks=sinks,
                                  query_start_loc=torch.from_numpy(st).cuda(), max_query_len=max(qs))
        close(out, exact, size, "bf16", 200)
        assert fd.device_status() == 0


def test_window_bad_page_inside_is_masked_and_reported():
    import flashdec_b200 as fd
    from flashdec_b200 import _lib

    for qs in ([1], [3], [150]):
        c = Cache(4, [200], bs=16)
        q, qn = c.queries(qs[0], 8)
        table, keys = c.table.clone(), np.arange(200)
        table[0, 10] = c.pool
        fd.device_status(clear=True)
        out = fd.window_attention(q, c.k, c.v, table, c.seq, window=90, sinks=3,
                                  query_start_loc=torch.tensor([0] + qs, device="cuda"), max_query_len=qs[0])
        assert fd.device_status(clear=True) == _lib.FD_STATUS_BAD_BLOCK_ID
        mask = ref.window_mask(200, qs[0], 90, 3) & (keys // 16 != 10)[None]
        for i in range(8):
            k, v = (ref._dense(x, c.table_np[0], 200)[:, i // 4] for x in (c.k_np, c.v_np))
            p = ref.softmax_rows(qn[:, i] @ k.T / np.sqrt(128), mask)
            close(out[:, i], p @ v, p @ np.abs(v), "bf16", 90)


def test_window_rows_without_a_key_are_zero():
    import flashdec_b200 as fd

    # three queries of which one is before the stream, an empty sequence, and
    # a long query range over few tokens
    for lens, qs in (([2, 0, 40], [3, 2, 4]), ([5, 130], [200, 130])):
        c = Cache(5, lens, fill=float("inf"))
        q, qn = c.queries(sum(qs), 16)
        out = fd.window_attention(q, c.k, c.v, c.table, c.seq, window=16, sinks=2,
                                  query_start_loc=torch.from_numpy(starts_of(qs)).cuda(),
                                  max_query_len=max(qs)).float().cpu().numpy()
        at = 0
        for n, ql in zip(lens, qs):
            blank = max(0, ql - n)
            assert (out[at:at + blank] == 0).all()
            assert np.isfinite(out[at:at + ql]).all()
            assert (out[at + blank:at + ql] != 0).any() or n == 0
            at += ql
    c = Cache(5, [0, 3])
    q, _ = c.queries(2, 16)
    out = fd.window_attention(q, c.k, c.v, c.table, c.seq, window=9)
    assert (out[0] == 0).all() and (out[1] != 0).any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("qs,hq,hkv", [([6], 8, 2), ([150], 8, 2), ([300], 16, 8), ([40], 2, 2)])
def test_window_masked_nonfinite_values_stay_out(bad, qs, hq, hkv):
    """K and V of one token are not finite: rows that do not see it are exact,
    rows that see it are not finite."""
    import flashdec_b200 as fd

    n, window, sinks = 400, 64, 3
    for token in (n - 2, n - qs[0], n - qs[0] - 20, 1):
        for where in ("v", "k"):
            c = Cache(6, [n], hkv=hkv, bs=16)
            q, qn = c.queries(qs[0], hq)
            blk, off = int(c.table_np[0, token // 16]), token % 16
            if where == "v":
                c.v[blk, :, off, 5] = bad
            else:
                c.k[blk, :, off] = bad if bad != bad else float("nan")
            out = fd.window_attention(q, c.k, c.v, c.table, c.seq, window=window, sinks=sinks,
                                      query_start_loc=torch.tensor([0] + qs, device="cuda"),
                                      max_query_len=qs[0])
            sees = ref.window_mask(n, qs[0], window, sinks)[:, token]
            exact, size = ref.window_attention_ref(qn, c.k_np, c.v_np, c.table_np, [n], window, sinks,
                                                   [0, qs[0]])
            if (~sees).any():
                close(out[torch.from_numpy(~sees).cuda()], exact[~sees], size[~sees], "bf16", 70)
            got = out.float().cpu().numpy()[sees]
            if where == "v":
                assert not np.isfinite(got[:, :, 5]).any()
                rest = np.delete(got, 5, axis=2)
                assert np.isfinite(rest).all()
            else:
                assert not np.isfinite(got).any()


def test_window_longer_than_any_sequence_is_the_decode():
    import flashdec_b200 as fd

    c = Cache(8, [1000, 77, 1], bs=32)
    q, _ = c.queries(3, 16)
    a = fd.window_attention(q, c.k, c.v, c.table, c.seq, window=1 << 40, sm_scale=0.2).float()
    b = fd.decode(q, c.k, c.v, c.table, c.seq, sm_scale=0.2).float()
    assert (a - b).abs().max() <= 2.0 ** -6  # two roundings of weights and output, |out| < 2


def test_window_out_strides_streams_and_longer_queries_than_announced():
    import flashdec_b200 as fd

    lens, qs = [300, 200], [40, 170]
    c = Cache(9, lens)
    q, qn = c.queries(210, 8)
    st = starts_of(qs)
    exact, size = ref.window_attention_ref(qn, c.k_np, c.v_np, c.table_np, lens, 50, 4, st)
    wide = torch.full((212, 8, 2, 131), 7.0, dtype=torch.bfloat16, device="cuda")
    out = wide[1:211, :, 1, 1:129]
    qv = torch.empty((210, 8, 256), dtype=torch.bfloat16, device="cuda")[:, :, ::2]
    qv.copy_(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fd.window_attention(qv, c.k, c.v, c.table, c.seq, window=50, sinks=4, out=out,
                                  query_start_loc=torch.from_numpy(st).cuda(), max_query_len=3)
    torch.cuda.current_stream().wait_stream(side)
    assert got.data_ptr() == out.data_ptr()
    close(out, exact, size, "bf16", 60)
    keep = torch.ones(wide.shape, dtype=torch.bool)
    keep[1:211, :, 1, 1:129] = False
    assert (wide.cpu()[keep] == 7).all()
    # rows no sequence owns are not written
    out2 = torch.full((214, 8, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    q2 = torch.cat([q[:2], q, q[:2]])
    fd.window_attention(q2, c.k, c.v, c.table, c.seq, window=50, sinks=4, out=out2,
                        query_start_loc=torch.from_numpy(st + 2).cuda(), max_query_len=170)
    assert (out2[:2] == 7).all() and (out2[212:] == 7).all()
    close(out2[2:212], exact, size, "bf16", 60)


def test_window_graph_replay():
    import flashdec_b200 as fd

    c = Cache(10, [900, 300])
    q, qn = c.queries(2, 16)
    fd.window_attention(q, c.k, c.v, c.table, c.seq, window=256, sinks=4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fd.window_attention(q, c.k, c.v, c.table, c.seq, window=256, sinks=4)
    for n in ([900, 300], [17, 1], [400, 299]):
        c.seq.copy_(torch.tensor(n))
        graph.replay()
        exact, size = ref.window_attention_ref(qn, c.k_np, c.v_np, c.table_np, n, 256, 4)
        close(out, exact, size, "bf16", 260)


def test_window_and_scored_batches_of_many_sequences():
    """More sequences than one launch takes, with empty and long ones among them."""
    import flashdec_b200 as fd

    rng = np.random.default_rng(21)
    lens = rng.integers(0, 24, 1100)
    lens[[0, 511, 512, 1099]] = [700, 0, 900, 300]
    lens = lens.tolist()
    c = Cache(20, lens, hkv=1, d=64, bs=8)
    q, qn = c.queries(len(lens), 2)
    out = fd.window_attention(q, c.k, c.v, c.table, c.seq, window=200, sinks=2)
    exact, size = ref.window_attention_ref(qn, c.k_np, c.v_np, c.table_np, lens, 200, 2)
    close(out, exact, size, "bf16", 202)
    scores = torch.ones((c.pool, 1, 8), device="cuda")
    out = fd.scored_decode(q, c.k, c.v, scores, c.table, c.seq)
    exact, size, want = ref.scored_decode_ref(qn, c.k_np, c.v_np, np.ones((c.pool, 1, 8)), c.table_np, lens)
    close(out, exact, size, "bf16", 900)
    assert (np.abs(scores.double().cpu().numpy() - want) <= 1e-4 * np.abs(want - 1) + 1e-6).all()
    qs = [min(n, 3) for n in lens]
    q, qn = c.queries(sum(qs), 2)
    st = starts_of(qs)
    out = fd.window_attention(q, c.k, c.v, c.table, c.seq, window=30, sinks=1, max_query_len=3,
                              query_start_loc=torch.from_numpy(st).cuda())
    exact, size = ref.window_attention_ref(qn, c.k_np, c.v_np, c.table_np, lens, 30, 1, st)
    close(out, exact, size, "bf16", 31)


SCORED = [
    ("bf16", 16, 2, 128, 32, "planes", [1, 2, 33, 300]),
    ("fp16", 32, 8, 128, 16, "nhd", [700, 5, 0, 64]),
    ("bf16", 8, 8, 64, 8, "planes", [1, 9, 200]),
    ("fp16", 7, 1, 64, 8, "dims", [150]),
    ("bf16", 40, 2, 128, 32, "odd", [130, 64]),
    ("bf16", 5, 1, 128, 16, "planes", [5000]),
    ("bf16", 64, 1, 128, 16, "planes", [2100, 3]),
]


@pytest.mark.parametrize("case", SCORED, ids=[f"s{i}" for i in range(len(SCORED))])
def test_scored_decode(case):
    import flashdec_b200 as fd

    dtype, hq, hkv, d, bs, layout, lens = case
    c = Cache(11, lens, dtype=dtype, hkv=hkv, d=d, bs=bs, layout=layout, fill=float("nan"))
    q, qn = c.queries(len(lens), hq, 1.5)
    start = np.abs(c.rng.standard_normal((c.pool, hkv, bs))).astype(np.float32)
    for b, n in enumerate(lens):  # the newest token's slot holds garbage
        if n:
            start[c.table_np[b, (n - 1) // bs], :, (n - 1) % bs] = np.nan
    store = torch.full((c.pool, bs, hkv + 1), -3.0, device="cuda")
    scores = store.permute(0, 2, 1)[:, :hkv] if layout == "nhd" else torch.empty(start.shape, device="cuda")
    scores.copy_(torch.from_numpy(start))
    fd.device_status(clear=True)
    out = fd.scored_decode(q, c.k, c.v, scores, c.table, c.seq)
    exact, size, want = ref.scored_decode_ref(qn, c.k_np, c.v_np, start, c.table_np, lens)
    close(out, exact, size, dtype, max(lens))
    got = scores.double().cpu().numpy()
    base = np.where(np.isnan(start), 0.0, start)
    assert not np.isnan(got).any()
    assert (np.abs(got - want) <= 1e-4 * (want - base) + 1e-6 * base + 1e-9).all()
    assert fd.device_status() == 0
    # the weights of each query head sum to one
    assert np.allclose((got - base).sum(), sum(n > 0 for n in lens) * hq, rtol=1e-4)


def test_scored_decode_is_deterministic_and_accumulates():
    import flashdec_b200 as fd

    c = Cache(12, [3000, 1500, 37], bs=32)
    q, _ = c.queries(3, 16)
    runs = []
    for _ in range(2):
        s = torch.zeros((c.pool, 2, 32), device="cuda")
        outs = [fd.scored_decode(q, c.k, c.v, s, c.table, c.seq) for _ in range(3)]
        assert torch.equal(outs[0], outs[2])
        runs.append(s)
    assert torch.equal(*runs)
    once = torch.zeros_like(runs[0])
    fd.scored_decode(q, c.k, c.v, once, c.table, c.seq)
    three = once * 3
    for b, n in enumerate(c.lens):  # the newest token is set each time
        at = (int(c.table_np[b, (n - 1) // 32]), slice(None), (n - 1) % 32)
        three[at] = once[at]
    assert torch.allclose(runs[0], three, rtol=1e-6, atol=0)


def test_scored_decode_of_nan_and_infinite_keys():
    import flashdec_b200 as fd

    c = Cache(13, [100, 100])
    c.k[int(c.table_np[0, 2]), 1, 3] = float("nan")
    q, qn = c.queries(2, 8)
    scores = torch.zeros((c.pool, 2, 16), device="cuda")
    out = fd.scored_decode(q, c.k, c.v, scores, c.table, c.seq)
    assert torch.isnan(out[0, 4:]).all()
    assert torch.isfinite(out[0, :4]).all() and torch.isfinite(out[1]).all()
    live = torch.isnan(scores).flatten(2).any(-1)
    assert set(map(tuple, torch.nonzero(live).tolist())) == {(int(x), 1) for x in c.table_np[0, :7]}


EVICT = [
    # dtype, hkv, d, bs, layout, lens, budget, sinks, recent
    ("bf16", 2, 128, 32, "planes", [100, 33, 1, 64], 64, 4, 16),
    ("fp16", 8, 64, 16, "nhd", [300, 299, 17], 96, 0, 0),
    ("bf16", 3, 128, 8, "dims", [70, 9], 9, 4, 5),
    ("fp16", 1, 128, 16, "odd", [2500, 64, 0], 1000, 1, 333),
    ("bf16", 2, 64, 8, "planes", [1030, 1025, 1024], 1024, 7, 100),
    ("bf16", 1, 64, 32, "planes", [40], 1, 0, 0),
    ("bf16", 1, 64, 32, "planes", [40], 1, 0, 1),
]


@pytest.mark.parametrize("case", EVICT, ids=[f"e{i}" for i in range(len(EVICT))])
@pytest.mark.parametrize("values", ["ties", "random", "special"])
def test_evict_tokens(case, values):
    import flashdec_b200 as fd

    dtype, hkv, d, bs, layout, lens, budget, sinks, recent = case
    new = [-(-min(n, budget) // bs) for n in lens]
    c = Cache(14, lens, dtype=dtype, hkv=hkv, d=d, bs=bs, layout=layout, extra_pages=sum(new),
              index=torch.int64 if layout == "nhd" else torch.int32)
    w = np.exp(2 * c.rng.standard_normal((c.pool, hkv, bs))).astype(np.float32)
    if values == "ties":
        w = np.round(w)
    elif values == "special":
        pick = c.rng.integers(0, 8, w.shape)
        for i, x in enumerate((0.0, -0.0, np.nan, np.inf, -np.inf, -1.5, 1e-42)):
            w[pick == i] = x
    table = np.full((len(lens), max(max(new), 1) + 1), -1, np.int64)
    at = 0
    for b, m in enumerate(new):
        table[b, :m] = c.spare[at:at + m]
        at += m
    scores = torch.from_numpy(w).cuda()
    fd.device_status(clear=True)
    kept, left = fd.evict_tokens(c.k, c.v, scores, c.table, c.seq, torch.from_numpy(table).cuda(),
                                 budget=budget, sinks=sinks, recent=recent)
    want = ref.evict_tokens_ref(c.k_np, c.v_np, w, c.table_np, lens, table, budget, sinks, recent)
    assert left.dtype == c.seq.dtype and left.tolist() == list(want[1])
    assert kept.dtype == torch.int32 and np.array_equal(kept.cpu().numpy(), want[0])
    for got, exp in zip((c.k, c.v, scores), want[2:]):
        assert np.array_equal(got.double().cpu().numpy(), exp.astype(np.float64), equal_nan=True)
    assert fd.device_status() == 0


def test_evict_bad_pages_are_skipped_and_reported():
    import flashdec_b200 as fd
    from flashdec_b200 import _lib

    c = Cache(15, [64], extra_pages=2)
    scores = torch.rand((c.pool, 2, 16), device="cuda")
    before = c.k.clone()
    fd.device_status(clear=True)
    fd.evict_tokens(c.k, c.v, scores, c.table, c.seq, torch.tensor([[c.pool, -1]], device="cuda"), budget=32)
    assert fd.device_status(clear=True) == _lib.FD_STATUS_BAD_BLOCK_ID
    assert torch.equal(c.k, before)


def test_refusals():
    import flashdec_b200 as fd

    c = Cache(16, [64, 30], extra_pages=4)
    q, _ = c.queries(2, 8)
    scores = torch.zeros((c.pool, 2, 16), device="cuda")
    st = torch.tensor([0, 1, 2], device="cuda")
    good = dict(q=q, k_cache=c.k, v_cache=c.v, block_tables=c.table, seq_lens=c.seq, window=4)

    def refuse(match, **change):
        with pytest.raises(ValueError, match=match):
            fd.window_attention(**{**good, **change})

    fd.window_attention(**good)
    refuse("window", window=0)
    refuse("sinks", sinks=-1)
    refuse("kv_layout", kv_layout="blocked")
    refuse("same dtype", q=q.half())
    refuse("device", q=q.cpu())
    refuse("CUDA", k_cache=c.k.cpu())
    refuse("shape", q=q[0])
    refuse("head_dim", q=q[..., :64])
    refuse("num_q_heads", q=q[:, :7])
    refuse("4D", k_cache=c.k[0], v_cache=c.v[0])
    refuse("same shape", v_cache=c.v[:-1])
    refuse("float16 or bfloat16", q=q.float(), k_cache=c.k.float(), v_cache=c.v.float())
    refuse("block_size", k_cache=c.k[:, :, :5], v_cache=c.v[:, :, :5])
    refuse("int32 or int64", block_tables=c.table.short())
    refuse("int32 or int64", seq_lens=c.seq.float())
    refuse("one row/value", seq_lens=c.seq[:1])
    refuse("one row per sequence", q=q[:1])
    refuse("max_query_len", query_start_loc=st)
    refuse("max_query_len", query_start_loc=st, max_query_len=0)
    refuse("max_query_len", max_query_len=2)
    refuse("num_seqs", query_start_loc=st[:2], max_query_len=1)
    refuse("out must", out=torch.empty_like(q, dtype=torch.float32))
    refuse("out must", out=torch.empty_like(q[:1]))
    refuse("max_blocks", block_tables=c.table[:, :0])

    with pytest.raises(ValueError, match="scores must have shape"):
        fd.scored_decode(q, c.k, c.v, scores[:, :1], c.table, c.seq)
    with pytest.raises(ValueError, match="float32"):
        fd.scored_decode(q, c.k, c.v, scores.double(), c.table, c.seq)
    with pytest.raises(ValueError, match="one row per sequence"):
        fd.scored_decode(q[:1], c.k, c.v, scores, c.table, c.seq)

    new = torch.zeros((2, 2), dtype=torch.int32, device="cuda")
    for match, kw in (("budget", dict(budget=0)), ("negative", dict(budget=8, sinks=-1)),
                      ("exceed", dict(budget=8, sinks=4, recent=5)),
                      ("cannot hold", dict(budget=33))):
        with pytest.raises(ValueError, match=match):
            fd.evict_tokens(c.k, c.v, scores, c.table, c.seq, new, **kw)
    with pytest.raises(ValueError, match="new_block_tables"):
        fd.evict_tokens(c.k, c.v, scores, c.table, c.seq, new[0], budget=8)
    # an empty batch is no error
    none = c.table[:0], c.seq[:0]
    assert fd.window_attention(q[:0], c.k, c.v, *none, window=3).shape == (0, 8, 128)
    assert fd.scored_decode(q[:0], c.k, c.v, scores, *none).shape == (0, 8, 128)
    kept, left = fd.evict_tokens(c.k, c.v, scores, *none, new[:0], budget=8)
    assert kept.shape == (0, 2, 8) and left.shape == (0,)
