"""Workloads of the bounded-cache operators: windowed attention with sink
tokens, decode attention that accumulates each cached token's attention
weight, and eviction of the least attended tokens.

Every case runs in two forms: elementary torch operations in 32 bits
(``own = False``) and the package's operators (``own = True``), on the same
inputs.  ``exact`` is the operators' definition in 64 bits.
"""

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _window(name, *, dtype, hq, hkv, d, bs, batch, ctx, q, window, sinks, layout="planes"):
    return {"name": name, "op": "window", "dtype": dtype, "hq": hq, "hkv": hkv, "d": d, "bs": bs,
            "batch": batch, "ctx_lo": ctx[0], "ctx_hi": ctx[1], "q_lo": q[0], "q_hi": q[1],
            "window": window, "sinks": sinks, "layout": layout}


def _scored(name, *, dtype, hq, hkv, d, bs, batch, ctx, layout="planes"):
    return {"name": name, "op": "scored", "dtype": dtype, "hq": hq, "hkv": hkv, "d": d, "bs": bs,
            "batch": batch, "ctx_lo": ctx[0], "ctx_hi": ctx[1], "layout": layout}


def _evict(name, *, dtype, hkv, d, bs, batch, ctx, budget, sinks, recent, layout="planes"):
    return {"name": name, "op": "evict", "dtype": dtype, "hkv": hkv, "d": d, "bs": bs,
            "batch": batch, "ctx_lo": ctx[0], "ctx_hi": ctx[1], "budget": budget, "sinks": sinks,
            "recent": recent, "layout": layout}


def listed():
    """Head layouts: 16/2 heads of 128 with 32-token pages (the Qwen2.5-3B
    shape), 32/8 heads of 128 with 16-token pages (the Llama-3-8B shape), and
    smaller ones with 64-dim heads."""
    return [
        # one chat session, one new token: the launch is the cost
        _window("window_one_token", dtype="bf16", hq=16, hkv=2, d=128, bs=32, batch=1,
                ctx=(2048, 2048), q=(1, 1), window=1024, sinks=4),
        # a serving batch of long sessions, one new token each
        _window("window_batch64", dtype="bf16", hq=32, hkv=8, d=128, bs=16, batch=64,
                ctx=(512, 131072), q=(1, 1), window=4096, sinks=4),
        # ragged drafts of a speculative step, verified in one call (vLLM page layout)
        _window("window_drafts", dtype="fp16", hq=16, hkv=4, d=64, bs=16, batch=24,
                ctx=(300, 9000), q=(1, 7), window=1500, sinks=1, layout="nhd"),
        # one long prompt chunk at the end of an 8k context
        _window("window_prompt_8k", dtype="bf16", hq=32, hkv=8, d=128, bs=16, batch=1,
                ctx=(8192, 8192), q=(8192, 8192), window=2048, sinks=4),
        # a ragged batch of odd prompt chunks, some shorter than the window
        _window("window_prompts_ragged", dtype="fp16", hq=16, hkv=2, d=128, bs=32, batch=6,
                ctx=(700, 5003), q=(65, 2001), window=1000, sinks=8),
        # one session with scores kept: the launch is the cost
        _scored("scored_one_token", dtype="bf16", hq=16, hkv=2, d=128, bs=32, batch=1,
                ctx=(1024, 1024)),
        # the uniform decode batch of the package's main benchmark
        _scored("scored_batch8", dtype="bf16", hq=16, hkv=2, d=128, bs=32, batch=8,
                ctx=(2048, 2048)),
        # ragged long sessions
        _scored("scored_ragged24", dtype="fp16", hq=32, hkv=8, d=128, bs=16, batch=24,
                ctx=(512, 32768), layout="nhd"),
        # one very long session
        _scored("scored_long", dtype="bf16", hq=32, hkv=8, d=128, bs=16, batch=1,
                ctx=(131071, 131071)),
        # one session trimmed back to its budget
        _evict("evict_one", dtype="bf16", hkv=2, d=128, bs=32, batch=1, ctx=(1088, 1088),
               budget=1024, sinks=4, recent=256),
        # the steady state of a batch: a few hundred tokens over the budget each
        _evict("evict_steady", dtype="bf16", hkv=8, d=128, bs=16, batch=16, ctx=(4097, 4480),
               budget=4096, sinks=4, recent=1024, layout="nhd"),
        # long prompts cut down to their budget
        _evict("evict_prompts", dtype="fp16", hkv=8, d=128, bs=16, batch=6, ctx=(9001, 65536),
               budget=4000, sinks=4, recent=512),
    ]


def _spread(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm, odd ones among them."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    n = min(hi, max(lo, n))
    return n + 1 if n == 3072 else n


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(("window", "window", "window", "scored", "scored", "evict", "evict"))
        hkv = rng.choice((1, 2, 4, 8))
        c = {"op": op, "dtype": rng.choice(("bf16", "fp16")), "hq": hkv * rng.choice((1, 2, 4, 5, 7, 8)),
             "hkv": hkv, "d": rng.choice((64, 128, 128)), "bs": rng.choice((8, 16, 32)),
             "layout": rng.choice(("planes", "nhd"))}
        hi = _spread(rng, 256, 131072)
        lo = _spread(rng, min(hi, max(64, hi // 16)), hi)
        c["batch"] = _spread(rng, 1, max(1, min(64, 1500000 // hi)))
        if op == "window":
            c["window"], c["sinks"] = _spread(rng, 64, 4096), rng.choice((0, 1, 4, 16, 37))
            form = rng.choice(("token", "drafts", "prompts"))
            q_hi = {"token": 1, "drafts": _spread(rng, 2, 16), "prompts": _spread(rng, 100, 4096)}[form]
            if form == "prompts":
                hi = min(hi, 16384)
                lo = min(lo, hi)
                c["batch"] = min(c["batch"], 8)
            q_hi = min(q_hi, lo)
            c["q_lo"], c["q_hi"] = _spread(rng, max(1, q_hi // 8), q_hi), q_hi
        if op == "evict":
            del c["hq"]
            c["budget"] = _spread(rng, max(32, hi // 16), hi)
            c["sinks"] = rng.choice((0, 4, 7)) if c["budget"] > 16 else 0
            c["recent"] = rng.randrange(0, c["budget"] // 2)
        c["ctx_lo"], c["ctx_hi"] = lo, hi
        if _cost(c) <= most and _plain_elements(c) <= 1 << 31:
            return c


def _lens(case):
    """Context lengths of a case: the longest first, the others spread between
    ctx_lo and ctx_hi over their logarithm."""
    rng = random.Random(case["ctx_hi"] * 131 + case["batch"])
    return [case["ctx_hi"]] + [_spread(rng, case["ctx_lo"], case["ctx_hi"])
                               for _ in range(case["batch"] - 1)]


def _query_lens(case):
    """Query tokens of each sequence (at most its length), spread like the lengths."""
    rng = random.Random(case["q_hi"] * 137 + case["batch"])
    return [min(n, _spread(rng, case["q_lo"], case["q_hi"]) if b else case["q_hi"])
            for b, n in enumerate(_lens(case))]


def _visible(n, q, window, sinks):
    """(query, key) pairs that see each other, and the distinct keys seen, of
    a sequence of n tokens whose last q are the queries."""
    pairs, first = 0, n - q
    # position p sees min(p + 1, window) recent keys and the sinks before them
    full = max(0, n - max(first, window - 1))  # queries whose window is full
    pairs += full * window
    part = q - full
    pairs += part * (first + 1) + part * (part - 1) // 2
    lo = max(0, first - window + 1)
    if sinks:
        # the queries at p >= window miss the keys before p - window + 1
        a, b = max(first, window), n - 1  # missing min(sinks, p - window + 1) sinks each
        if b >= a:
            x, y = a - window + 1, b - window + 1
            ramp = max(0, min(y, sinks) - x + 1)
            pairs += ramp * x + ramp * (ramp - 1) // 2 + (y - x + 1 - ramp) * sinks
    return pairs, (n - lo) + min(sinks, lo)


def work(case):
    """Bytes: each visible K and V row, q, out, block-table entry and length
    once (and the scores read and written).  Flops: the two products."""
    lens, row = _lens(case), case["d"] * 2
    pages = sum(-(-n // case["bs"]) for n in lens)
    if case["op"] == "window":
        qs = _query_lens(case)
        seen = [_visible(n, q, case["window"], case["sinks"]) for n, q in zip(lens, qs)]
        kv = sum(k for _, k in seen) * case["hkv"] * row * 2
        io = 2 * sum(qs) * case["hq"] * row
        table = sum(-(-k // case["bs"]) for _, k in seen) * 4
        return {"bytes": kv + io + table + 8 * len(lens),
                "flops": 4 * case["d"] * case["hq"] * sum(p for p, _ in seen)}
    if case["op"] == "scored":
        total = sum(lens)
        return {"bytes": total * case["hkv"] * (2 * row + 8) + 2 * len(lens) * case["hq"] * row
                + 4 * pages + 4 * len(lens),
                "flops": 4 * case["d"] * case["hq"] * total}
    kept = sum(min(n, case["budget"]) for n in lens)
    return {"bytes": case["hkv"] * (4 * sum(lens) + kept * (4 * row + 8)) + 8 * pages, "flops": 0}


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def _plain_elements(case):
    """The plain form's largest tensor, in elements."""
    if case["op"] == "evict":
        return case["batch"] * min(case["budget"], case["ctx_hi"]) * case["hkv"] * case["d"]
    if case["op"] == "scored":
        return case["batch"] * case["ctx_hi"] * case["hkv"] * max(case["d"], case["hq"] // case["hkv"])
    keys = _key_columns(case)
    return case["batch"] * keys * max(case["hkv"] * case["d"], case["hq"] * case["q_hi"])


def _key_columns(case):
    return min(case["ctx_hi"], case["sinks"] + case["window"] + case["q_hi"] - 1)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _pages(lens, bs, gen, spare=0):
    """A scattered block table [batch, pages of the longest] (-1 beyond a
    sequence's pages) over a pool with some pages to spare."""
    counts = [-(-n // bs) for n in lens]
    pool = sum(counts) + max(4, sum(counts) // 8) + spare
    perm = torch.randperm(pool, generator=gen, device="cuda")
    table = torch.full((len(lens), max(counts)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, perm[at:], pool


def _pool(case, blocks, gen):
    """K and V caches [blocks, hkv, bs, d] of unit normal values: two planes, or
    views of one [blocks, 2, bs, hkv, d] allocation."""
    shape = (blocks, case["hkv"], case["bs"], case["d"])
    dtype = _DTYPES[case["dtype"]]
    if case["layout"] == "planes":
        k, v = (torch.empty(shape, dtype=dtype, device="cuda") for _ in range(2))
        return k.normal_(generator=gen), v.normal_(generator=gen)
    kv = torch.empty((blocks, 2, case["bs"], case["hkv"], case["d"]), dtype=dtype, device="cuda")
    kv.normal_(generator=gen)
    return kv[:, 0].permute(0, 2, 1, 3), kv[:, 1].permute(0, 2, 1, 3)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    lens = _lens(case)
    new = [-(-min(n, case["budget"]) // case["bs"]) for n in lens] if case["op"] == "evict" else []
    table, spare, pool = _pages(lens, case["bs"], gen, sum(new))
    k, v = _pool(case, pool, gen)
    s = {"case": case, "k": k, "v": v, "block_tables": table,
         "seq_lens": torch.tensor(lens, dtype=torch.int32, device="cuda")}
    dtype = _DTYPES[case["dtype"]]
    if case["op"] == "window":
        qs = _query_lens(case)
        starts = [0]
        for n in qs:
            starts.append(starts[-1] + n)
        s["q"] = torch.randn((starts[-1], case["hq"], case["d"]), generator=gen, device="cuda",
                             dtype=torch.float32).mul_(1.5).to(dtype)
        s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        # row of q (or the pad row) of each sequence's i-th query of q_hi
        at = torch.arange(case["q_hi"], device="cuda")[None] + s["starts"][:-1, None]
        s["query_rows"] = torch.where(at < s["starts"][1:, None], at, starts[-1])
        owner = [b for b, n in enumerate(qs) for _ in range(n)]
        s["owner"] = torch.tensor(owner, device="cuda")
        return s
    shape = (pool, case["hkv"], case["bs"])
    if case["op"] == "scored":
        s["q"] = torch.randn((len(lens), case["hq"], case["d"]), generator=gen, device="cuda",
                             dtype=torch.float32).mul_(1.5).to(dtype)
        s["scores"] = torch.rand(shape, generator=gen, device="cuda").square_().mul_(4)
        return s
    # accumulated weights: a few heavy tokens, many light ones, ties among them
    w = torch.randn(shape, generator=gen, device="cuda").mul_(2).exp_().mul_(0.01)
    coarse = torch.rand(shape, generator=gen, device="cuda") < 0.25
    s["scores"] = torch.where(coarse, torch.round(w * 64) / 64, w)
    s["new_tables"] = torch.full((len(lens), max(new)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(new):
        s["new_tables"][b, :n] = spare[at:at + n]
        at += n
    return s


# ---------------------------------------------------------------------------
# the operators: the package's, and their plain form
# ---------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if own:
        import flashdec_b200 as fd

        if c["op"] == "window":
            return fd.window_attention(s["q"], s["k"], s["v"], s["block_tables"], s["seq_lens"],
                                       window=c["window"], sinks=c["sinks"],
                                       query_start_loc=s["starts"] if c["q_hi"] > 1 else None,
                                       max_query_len=c["q_hi"])
        if c["op"] == "scored":
            out = fd.scored_decode(s["q"], s["k"], s["v"], s["scores"], s["block_tables"],
                                   s["seq_lens"])
            return out, s["scores"]
        kept, lens = fd.evict_tokens(s["k"], s["v"], s["scores"], s["block_tables"], s["seq_lens"],
                                     s["new_tables"], budget=c["budget"], sinks=c["sinks"],
                                     recent=c["recent"])
        return kept, lens, s["scores"], s["k"], s["v"]
    return {"window": _plain_window, "scored": _plain_scored, "evict": _plain_evict}[c["op"]](s)


def _rows(cache, tables, tokens, bs):
    """Cache rows [batch, tokens, heads, ...] of the token positions
    [batch, n]; a position without a page reads page 0."""
    page = tables.gather(1, torch.clamp(tokens // bs, max=tables.shape[1] - 1)).clamp(min=0).long()
    return cache[page, :, tokens % bs]


def _plain_window(s):
    c = s["case"]
    batch, hkv, hq, d, bs = c["batch"], c["hkv"], c["hq"], c["d"], c["bs"]
    n = s["seq_lens"].long()[:, None]
    first = n - (s["starts"][1:] - s["starts"][:-1]).long()[:, None]  # position of the first query
    # the keys any of a sequence's queries sees: sinks, then the window's span
    lo = torch.clamp(first - c["window"] + 1, min=0)
    sinks = torch.clamp(lo, max=c["sinks"])
    col = torch.arange(_key_columns(c), device="cuda")[None]
    key = torch.where(col < sinks, col, lo + col - sinks)
    real = key < n
    key = torch.where(real, key, 0)
    k = _rows(s["k"], s["block_tables"], key, bs).float()
    v = _rows(s["v"], s["block_tables"], key, bs).float()
    q = torch.cat([s["q"], s["q"].new_zeros(1, hq, d)])[s["query_rows"]].float()
    q = q.view(batch, c["q_hi"], hkv, hq // hkv, d).permute(0, 2, 3, 1, 4)
    q = q.reshape(batch, hkv, -1, d)
    p = torch.matmul(q, k.permute(0, 2, 3, 1)).mul_(1.0 / math.sqrt(d))
    pos = (first + torch.arange(c["q_hi"], device="cuda")[None])[:, :, None]
    key, real = key[:, None], real[:, None]
    see = real & (key <= pos) & ((key > pos - c["window"]) | (key < c["sinks"])) & (pos >= 0)
    see = see[:, None, None].expand(batch, 1, hq // hkv, c["q_hi"], -1).reshape(batch, 1, -1, see.shape[-1])
    p.masked_fill_(~see, -math.inf)
    p.sub_(p.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v.permute(0, 2, 1, 3)) / total.clamp(min=1e-30)
    o = o.view(batch, hkv, hq // hkv, c["q_hi"], d).permute(0, 3, 1, 2, 4).reshape(batch, c["q_hi"], hq, d)
    at = torch.arange(s["q"].shape[0], device="cuda") - s["starts"][s["owner"]]
    return o[s["owner"], at].to(s["q"].dtype)


def _plain_scored(s):
    c = s["case"]
    batch, hkv, hq, d, bs = c["batch"], c["hkv"], c["hq"], c["d"], c["bs"]
    n = s["seq_lens"].long()[:, None]
    tok = torch.arange(c["ctx_hi"], device="cuda")[None].expand(batch, -1)
    real = tok < n
    k = _rows(s["k"], s["block_tables"], tok, bs).float()
    q = s["q"].float().view(batch, hkv, hq // hkv, d)
    p = torch.matmul(q, k.permute(0, 2, 3, 1)).mul_(1.0 / math.sqrt(d))
    del k
    p.masked_fill_(~real[:, None, None], -math.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    v = _rows(s["v"], s["block_tables"], tok, bs).float()
    out = torch.matmul(p, v.permute(0, 2, 1, 3)).view(batch, hq, d).to(s["q"].dtype)
    # the newest token's score starts here; the others are added to
    page = s["block_tables"].gather(1, torch.clamp(tok // bs, max=s["block_tables"].shape[1] - 1))
    page = page.clamp(min=0).long()
    flat = s["scores"].view(-1)
    heads = torch.arange(hkv, device="cuda")[None, :, None]
    slot = (page[:, None] * hkv + heads) * bs + (tok % bs)[:, None]
    last = slot.gather(2, (n - 1)[:, None].expand(-1, hkv, 1)).reshape(-1)
    flat[last] = 0.0
    add = torch.where(real[:, None], p.sum(2), 0.0)
    flat.index_add_(0, torch.where(real[:, None], slot, 0).reshape(-1), add.reshape(-1))
    return out, s["scores"]


def _plain_evict(s):
    c = s["case"]
    hkv, bs, budget = c["hkv"], c["bs"], c["budget"]
    n = s["seq_lens"].long()[:, None]
    tok = torch.arange(c["ctx_hi"], device="cuda")[None].expand(c["batch"], -1)
    w = _rows(s["scores"], s["block_tables"], tok, bs).permute(0, 2, 1)  # [batch, heads, tokens]
    safe = ((tok < c["sinks"]) | (tok >= n - c["recent"])) & (tok < n)
    w = torch.where(safe[:, None], math.inf, w)
    w = torch.where((tok < n)[:, None], w, -1.0)
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices[:, :, :budget]
    left = torch.clamp(n, max=budget)
    rank = torch.arange(order.shape[2], device="cuda")[None]
    order = torch.where((rank < left)[:, None], order, c["ctx_hi"]).sort(dim=-1).values
    kept = torch.full((c["batch"], hkv, budget), -1, dtype=torch.int32, device="cuda")
    kept[:, :, :order.shape[2]] = torch.where((rank < left)[:, None], order, -1).int()
    # rows beyond a sequence's new length repeat its first row's copy
    order = torch.where((rank < left)[:, None], order, order[:, :, :1])
    to = torch.where(rank < left, rank, 0)[:, None].expand(-1, hkv, -1)
    heads = torch.arange(hkv, device="cuda")[None, :, None]
    src = s["block_tables"][:, None].expand(-1, hkv, -1).gather(2, order // bs).long()
    dst = s["new_tables"][:, None].expand(-1, hkv, -1).gather(2, to // bs).long()
    s["k"][dst, heads, to % bs] = s["k"][src, heads, order % bs]
    s["v"][dst, heads, to % bs] = s["v"][src, heads, order % bs]
    s["scores"][dst, heads, to % bs] = s["scores"][src, heads, order % bs]
    return kept, left[:, 0].int(), s["scores"], s["k"], s["v"]


# ---------------------------------------------------------------------------
# the definition in 64 bits, one sequence and KV head at a time
# ---------------------------------------------------------------------------
def _dense(cache, table, h, n):
    """The first n rows of KV head h of one sequence, contiguous."""
    bs = cache.shape[2]
    return cache[table[:-(-n // bs)].long(), h].reshape(-1, *cache.shape[3:])[:n]


def exact(case, seed):
    s = prepare(case, seed)
    lens, g = s["seq_lens"].tolist(), case.get("hq", 0) // case["hkv"]
    if case["op"] == "evict":
        return _exact_evict(case, s, lens)
    scale = 1.0 / math.sqrt(case["d"])
    starts = s["starts"].tolist() if case["op"] == "window" else list(range(len(lens) + 1))
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    scores = s["scores"].double() if case["op"] == "scored" else None
    for b, n in enumerate(lens):
        table, (a, z) = s["block_tables"][b], starts[b:b + 2]
        pos = torch.arange(n - (z - a), n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")[None]
        hidden = key > pos
        if case["op"] == "window":
            hidden = hidden | ((key <= pos - case["window"]) & (key >= case["sinks"]))
        for h in range(case["hkv"]):
            k, v = (_dense(s[x], table, h, n).double() for x in ("k", "v"))
            mass = 0.0
            for i in range(h * g, h * g + g):
                x = (s["q"][a:z, i].double() @ k.T) * scale
                x[hidden.expand_as(x)] = -math.inf
                x = torch.softmax(x, dim=-1)
                out[a:z, i] = x @ v
                if scores is not None:
                    mass = mass + x.sum(0)
            if scores is not None:
                where = torch.arange(n, device="cuda")
                page = table[where // case["bs"]].long()
                old = scores[page, h, where % case["bs"]]
                old[-1] = 0.0
                scores[page, h, where % case["bs"]] = old + mass
    return out if scores is None else (out, scores)


def _exact_evict(case, s, lens):
    bs, budget = case["bs"], case["budget"]
    kept = torch.full((len(lens), case["hkv"], budget), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        m, table, new = min(n, budget), s["block_tables"][b], s["new_tables"][b]
        for h in range(case["hkv"]):
            w = _dense(s["scores"], table, h, n).double().cpu().numpy()
            if n <= budget:
                take = list(range(n))
            else:
                a, z = case["sinks"], n - case["recent"]
                mid = sorted(range(a, z), key=lambda t: -w[t])[:budget - a - case["recent"]]
                take = sorted(list(range(a)) + mid + list(range(z, n)))
            kept[b, h, :m] = torch.tensor(take, dtype=torch.int32)
            t = torch.tensor(take, device="cuda")
            j = torch.arange(m, device="cuda")
            for x in ("k", "v", "scores"):
                s[x][new[j // bs].long(), h, j % bs] = s[x][table[t // bs].long(), h, t % bs]
    return (kept, torch.tensor([min(n, budget) for n in lens], dtype=torch.int32),
            s["scores"], s["k"], s["v"])
