"""64-bit numpy statements of the bounded-cache operators (no counterpart in
the reference): windowed attention with sinks, decode with accumulated
attention weights, eviction by accumulated weight.  Caches are logical
[block, kv_head, token, dim]."""

from __future__ import annotations

import math

import numpy as np


def _dense(cache, row, n):
    """The first n tokens of one sequence: [n, heads, ...] (a page that is not
    in the cache reads as zeros)."""
    bs = cache.shape[2]
    out = np.zeros((n, cache.shape[1]) + cache.shape[3:], np.float64)
    for t in range(n):
        blk = int(row[t // bs])
        if 0 <= blk < cache.shape[0]:
            out[t] = cache[blk, :, t % bs]
    return out


def window_mask(n, q_len, window, sinks):
    """[q_len, n]: which keys the last q_len of n tokens see."""
    pos = np.arange(n - q_len, n)[:, None]
    key = np.arange(n)[None]
    return (key <= pos) & ((key > pos - window) | (key < sinks))


def softmax_rows(x, mask):
    """Softmax over the masked entries of each row; a row without one is zero."""
    x = np.where(mask, x, -np.inf)
    m = np.max(x, axis=-1, keepdims=True, initial=-np.inf)
    with np.errstate(invalid="ignore", over="ignore"):
        p = np.where(mask, np.exp(x - np.where(np.isneginf(m), 0.0, m)), 0.0)
    total = p.sum(-1, keepdims=True)
    return np.divide(p, total, out=np.zeros_like(p), where=total != 0)


def window_attention_ref(q, k_cache, v_cache, block_tables, seq_lens, window, sinks=0, starts=None,
                         sm_scale=None):
    """(out, mean |v|): the second is sum p |v|, the scale of its rounding."""
    hq, d = q.shape[1:]
    hkv = k_cache.shape[1]
    scale = 1.0 / math.sqrt(d) if sm_scale is None else sm_scale
    starts = range(len(seq_lens) + 1) if starts is None else starts
    out = np.zeros(q.shape, np.float64)
    size = np.zeros(q.shape, np.float64)
    for b, n in enumerate(seq_lens):
        a, z, n = int(starts[b]), int(starts[b + 1]), int(n)
        k, v = _dense(k_cache, block_tables[b], n), _dense(v_cache, block_tables[b], n)
        mask = window_mask(n, z - a, window, sinks)
        for i in range(hq):
            h = i // (hq // hkv)
            p = softmax_rows(q[a:z, i].astype(np.float64) @ k[:, h].T * scale, mask)
            # a weight of zero meets no value (0 * inf is not part of the sum)
            seen = mask.any(0)
            out[a:z, i] = p[:, seen] @ v[seen][:, h]
            size[a:z, i] = p[:, seen] @ np.abs(v[seen][:, h])
    return out, size


def scored_decode_ref(q, k_cache, v_cache, scores, block_tables, seq_lens, sm_scale=None):
    """(out, mean |v|, new scores)."""
    out, size = window_attention_ref(q, k_cache, v_cache, block_tables, seq_lens, 1 << 40,
                                     sm_scale=sm_scale)
    hq, d = q.shape[1:]
    hkv, bs = k_cache.shape[1:3]
    scale = 1.0 / math.sqrt(d) if sm_scale is None else sm_scale
    scores = scores.astype(np.float64).copy()
    for b, n in enumerate(seq_lens):
        n = int(n)
        k = _dense(k_cache, block_tables[b], n)
        for h in range(hkv):
            g = hq // hkv
            x = q[b, h * g:(h + 1) * g].astype(np.float64) @ k[:, h].T * scale
            w = softmax_rows(x, np.ones(x.shape, bool)).sum(0)
            for t in range(n):
                blk = int(block_tables[b][t // bs])
                if 0 <= blk < k_cache.shape[0]:
                    old = 0.0 if t == n - 1 else scores[blk, h, t % bs]
                    scores[blk, h, t % bs] = old + w[t]
    return out, size, scores


def evict_choice(weights, budget, sinks, recent):
    """Positions that stay, in order, of one (sequence, head)'s weights."""
    n = len(weights)
    if n <= budget:
        return list(range(n))
    mid = range(sinks, n - recent)

    def rank(t):  # NaN above every number, then the greater, then the earlier
        w = float(weights[t])
        return (0, 0.0, t) if math.isnan(w) else (1, -w + 0.0, t)

    best = sorted(mid, key=rank)[:budget - sinks - recent]
    return sorted(list(range(sinks)) + best + list(range(n - recent, n)))


def evict_tokens_ref(k_cache, v_cache, scores, block_tables, seq_lens, new_tables, budget, sinks=0,
                     recent=0):
    """(kept, new lengths, k, v, scores) with the new pages written."""
    hkv, bs = k_cache.shape[1:3]
    k, v, s = k_cache.copy(), v_cache.copy(), scores.copy()
    kept = np.full((len(seq_lens), hkv, budget), -1, np.int32)
    for b, n in enumerate(seq_lens):
        n = int(n)
        row = block_tables[b]
        for h in range(hkv):
            w = [scores[row[t // bs], h, t % bs] for t in range(n)]
            take = evict_choice(w, budget, sinks, recent)
            kept[b, h, :len(take)] = take
            for i, t in enumerate(take):
                for dst, src in ((k, k_cache), (v, v_cache), (s, scores)):
                    dst[new_tables[b][i // bs], h, i % bs] = src[row[t // bs], h, t % bs]
    return kept, np.minimum(seq_lens, budget), k, v, s
