"""window_attention where values are not finite and pages are not in the
cache: at lengths where a detour of its own would show, and element by element
against what the definition gives (a weight above 0 times an infinity is that
infinity, a weight of 0 times it NaN, opposite infinities NaN; a page that is
not in the cache holds no key).  Bounds as in test_bounded_cache_gpu.py."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import bounded_cache as ref  # noqa: E402
from tests.test_bounded_cache_gpu import Cache, U, starts_of  # noqa: E402

pytestmark = pytest.mark.gpu


def exact_rows(q, k, v, mask, scale):
    """(out, sum p |v|) of one head's rows: [rows, d], keys [n, d], [rows, n]."""
    with np.errstate(invalid="ignore"):
        p = ref.softmax_rows(q @ k.T * scale, mask)
    clean = np.where(np.isfinite(v), v, 0.0)
    out, size = p @ clean, p @ np.abs(clean)
    for t, e in zip(*np.nonzero(~np.isfinite(v))):
        with np.errstate(invalid="ignore"):
            out[:, e] = np.where(mask[:, t], out[:, e] + p[:, t] * v[t, e], out[:, e])
    return out, size


def compare(got, exact, size, dtype):
    assert np.array_equal(np.isnan(got), np.isnan(exact))
    assert np.array_equal(np.isinf(got), np.isinf(exact))
    inf = np.isinf(exact)
    assert (np.sign(got[inf]) == np.sign(exact[inf])).all()
    fine = np.isfinite(exact)
    bound = (2 * U[dtype] + 1e-4) * size + 1e-6
    assert (np.abs(got - exact)[fine] <= bound[fine]).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("what", ["nan", "inf", "first page", "page in the middle", "last page"])
def test_one_token_or_page_of_a_long_context(what, d):
    """768 queries of 8 heads over 200000 tokens, one value or page of which is
    bad: the rest of the batch and of the rows is exact, and no wait runs out."""
    import flashdec_b200 as fd
    from flashdec_b200 import _lib

    n, qs, group, bs = 200000, 768, 8, 16
    gen = torch.Generator(device="cuda").manual_seed(7)
    pages = n // bs
    k, v = (torch.randn((pages + 40, 1, bs, d), generator=gen, device="cuda").bfloat16() for _ in range(2))
    table = torch.full((2, pages), -1, dtype=torch.int32, device="cuda")
    table[0] = torch.randperm(pages, generator=gen, device="cuda")
    table[1, :40] = torch.arange(pages, pages + 40, device="cuda")
    lens = torch.tensor([n, 640], dtype=torch.int32, device="cuda")
    q = torch.randn((qs + 600, group, d), generator=gen, device="cuda").bfloat16()
    token, gone = n - 300, None
    if what in ("nan", "inf"):
        v[int(table[0, token // bs]), 0, token % bs, 3] = float(what)
    else:
        gone = {"first page": 0, "page in the middle": pages // 2, "last page": pages - 1}[what]
    asked = table.clone()
    if gone is not None:
        asked[0, gone] = 1 << 20
    fd.device_status(clear=True)
    out = fd.window_attention(q, k, v, asked, lens, window=n, max_query_len=qs,
                              query_start_loc=torch.tensor([0, qs, qs + 600], device="cuda"))
    torch.cuda.synchronize()
    assert fd.device_status(clear=True) == (0 if gone is None else _lib.FD_STATUS_BAD_BLOCK_ID)

    def check(rows, b, first, length):
        kk, vv = (x[table[b].long()[:length // bs]].reshape(length, d).double() for x in (k, v))
        odd = ~torch.isfinite(vv)
        vv[odd] = 0
        for r in rows:
            seen = torch.arange(length, device="cuda") <= first + r
            if gone is not None and b == 0:
                seen &= torch.arange(length, device="cuda") // bs != gone
            x = (q[b * qs + r].double() @ kk.T) / d ** 0.5
            p = torch.softmax(x.masked_fill(~seen, float("-inf")), -1)
            got, want, size = out[b * qs + r].double(), p @ vv, p @ vv.abs()
            if odd.any() and b == 0 and first + r >= token:
                hit = got[:, 3].clone()
                assert torch.isnan(hit).all() if what == "nan" else (hit == float("inf")).all()
                got[:, 3] = want[:, 3]
            assert ((got - want).abs() <= (2 * U["bf16"] + 1e-4) * size + 1e-6).all(), (b, r)

    check((0, 1, 255, 466, 467, 468, 469, 500, 767), 0, n - qs, n)
    check((0, 300, 599), 1, 40, 640)


FORMS = [
    # dtype, hq, hkv, d, bs, layout, length, queries, window, sinks
    ("bf16", 8, 2, 128, 16, "planes", 700, 300, 260, 20),
    ("bf16", 16, 2, 64, 32, "nhd", 900, 200, 700, 3),
    ("bf16", 4, 4, 128, 8, "planes", 650, 600, 150, 0),
    ("bf16", 5, 1, 64, 8, "nhd", 500, 500, 1000, 0),
    ("fp16", 8, 1, 128, 32, "planes", 600, 150, 200, 140),
    ("bf16", 8, 2, 128, 16, "planes", 700, 6, 260, 20),  # few rows: the other kernel
]


@pytest.mark.parametrize("form", FORMS, ids=[f"n{i}" for i in range(len(FORMS))])
@pytest.mark.parametrize("seed", range(4))
def test_every_element_is_what_the_definition_gives(form, seed):
    import flashdec_b200 as fd
    from flashdec_b200 import _lib

    dtype, hq, hkv, d, bs, layout, n, ql, window, sinks = form
    lens, qs = [n, 300], [ql, min(ql, 120)]
    c = Cache(50 + seed, lens, dtype=dtype, hkv=hkv, d=d, bs=bs, layout=layout)
    q, qn = c.queries(sum(qs), hq, 0.5)
    st = starts_of(qs)
    rng = np.random.default_rng(60 + seed)
    # infinities of both signs and NaN near the edges of what the rows see, the
    # same dimension hit more than once
    spots = [0, 1, sinks, n - ql - window + 1, n - window, n - ql, n - ql // 2, n - 1]
    spots = [t for t in spots if 0 <= t < n] + rng.integers(0, n, 3).tolist()
    for t in spots:
        x = (np.inf, -np.inf, np.nan)[rng.integers(0, 5) % 3]
        h, e = int(rng.integers(0, hkv)), int(rng.choice([0, 7, d - 1]))
        for b in range(1 if rng.integers(0, 2) else 2):
            if t < lens[b]:
                blk = int(c.table_np[b, t // bs])
                c.v[blk, h, t % bs, e] = x
                c.v_np[blk, h, t % bs, e] = x
    if seed == 1:  # a key whose score is -inf for the rows with a negative q there
        t = n - ql // 2
        blk = int(c.table_np[0, t // bs])
        c.k[blk, 0, t % bs, 2] = c.k_np[blk, 0, t % bs, 2] = np.inf
        q[:st[1], :hq // hkv, 2] = -q[:st[1], :hq // hkv, 2].abs() - 0.1
        qn = q.double().cpu().numpy()
        c.v[blk, 0, t % bs, 4] = c.v_np[blk, 0, t % bs, 4] = np.inf
    gone = {} if seed < 2 else {0: {0, n // bs // 2, (n - 1) // bs}, 1: {3}}
    table = c.table.clone()
    for b, pages in gone.items():
        for page in pages:
            table[b, page] = c.pool + page if page % 2 else -5
    wide = torch.full((sum(qs), hq, d + 3), 7.0, dtype=q.dtype, device="cuda")
    out = wide[..., 1:d + 1] if seed % 2 else torch.empty_like(q)
    fd.device_status(clear=True)
    fd.window_attention(q, c.k, c.v, table, c.seq, window=window, sinks=sinks, out=out,
                        query_start_loc=torch.from_numpy(st).cuda(), max_query_len=max(qs))
    status, told = fd.device_status(clear=True), False
    for b in range(2):
        mask = ref.window_mask(lens[b], qs[b], window, sinks)
        page = np.arange(lens[b]) // bs
        for g in gone.get(b, ()):
            told |= bool(mask[:, page == g].any())
            mask = mask & (page != g)[None]
        k, v = (ref._dense(x, c.table_np[b], lens[b]) for x in (c.k_np, c.v_np))
        for i in range(hq):
            h = i // (hq // hkv)
            exact, size = exact_rows(qn[st[b]:st[b + 1], i], k[:, h], v[:, h], mask, d ** -0.5)
            compare(out[st[b]:st[b + 1], i].double().cpu().numpy(), exact, size, dtype)
    assert status == (_lib.FD_STATUS_BAD_BLOCK_ID if told else 0)
    assert (wide[..., 0] == 7).all() and (wide[..., d + 1:] == 7).all()
