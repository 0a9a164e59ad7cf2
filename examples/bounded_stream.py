"""Streams longer than their cache: one attention layer served from a bounded
paged K/V cache.

Every stream's prompt goes through ``window_attention`` in chunks.  Then each
decoded token is rotated and appended (``fused_rope_kv_append``) and attends
to the whole cache through ``scored_decode``, which adds up the attention
weight of every cached token.  When a stream has outgrown its budget by
``slack`` tokens, ``evict_tokens`` moves the tokens worth keeping to fresh
pages and the old ones are freed, so the stream goes on for ever in
``budget + slack`` tokens of cache.

A prompt's tokens have no weights yet: their scores start at zero (their pages
may have been another stream's), and a prompt longer than the cache keeps the
sinks and its newest tokens.

    python examples/bounded_stream.py --streams 8 --prompt 5000 --tokens 600

Random weights stand for the model: q, k and v of each token are drawn, not
computed.  A token's rotary position is its position in the stream; its place
in the cache is another matter (keys are cached rotated).
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import flashdec_b200 as fd  # noqa: E402


class BoundedLayer:
    """The pages, block tables, lengths and scores of one layer's streams."""

    def __init__(self, streams, *, q_heads=16, kv_heads=2, head_dim=128, block_size=32, budget=2048,
                 slack=256, sinks=4, recent=512, dtype=torch.bfloat16, device="cuda"):
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.block_size, self.budget, self.slack = block_size, budget, slack
        self.sinks, self.recent = sinks, recent
        self.row = -(-(budget + slack) // block_size)  # pages of a stream at its longest
        kept = -(-budget // block_size)  # eviction of one stream needs that many more
        self.blocks = streams * self.row + kept
        shape = (self.blocks, kv_heads, block_size, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        self.scores = torch.zeros(shape[:3], device=device)
        self.free = list(range(self.blocks))
        self.pages = [[] for _ in range(streams)]
        self.length = [0] * streams  # cached tokens
        self.position = [0] * streams  # tokens of the stream so far
        self.evicted = 0

    def _tensor(self, rows, dtype=torch.int64):
        return torch.tensor(rows, dtype=dtype, device=self.k.device)

    def _table(self, streams):
        return self._tensor([self.pages[s] + [-1] * (self.row - len(self.pages[s])) for s in streams], torch.int32)

    def _slots(self, stream, tokens):
        """Pages and offsets of the stream's next `tokens` cache places."""
        start = self.length[stream]
        while len(self.pages[stream]) * self.block_size < start + tokens:
            self.pages[stream].append(self.free.pop())
        return self._places(stream, start, tokens)

    def _places(self, stream, start, tokens):
        places = range(start, start + tokens)
        return ([self.pages[stream][t // self.block_size] for t in places], [t % self.block_size for t in places])

    def append(self, streams, q, k, v, counts):
        """Rotate q and k, write k and v of each stream's next counts[i] tokens;
        returns the rotated q (rows in stream order)."""
        blocks, offsets, positions = [], [], []
        for s, n in zip(streams, counts):
            a, b = self._slots(s, n)
            blocks += a
            offsets += b
            positions += range(self.position[s], self.position[s] + n)
            self.length[s] += n
            self.position[s] += n
        return fd.fused_rope_kv_append(q, k, v, self.k, self.v, self._tensor(blocks), self._tensor(offsets),
                                       self._tensor(positions), rotary_dim=self.head_dim, base=1e6)

    def prompt(self, stream, q, k, v, chunk=1024):
        """A stream's prompt, windowed by its budget: chunk by chunk, the
        cache is cut back to the sinks and the newest before it overflows."""
        newest = self.budget - self.sinks
        outs = []
        for at in range(0, q.shape[0], chunk):
            n = min(chunk, q.shape[0] - at)
            step = 0
            while step < n:  # what fits the stream's pages goes in one call
                if self.length[stream] >= self.budget + self.slack:
                    self.evict([stream], newest)
                m = min(n - step, self.budget + self.slack - self.length[stream])
                part = slice(at + step, at + step + m)
                rot = self.append([stream], q[part], k[part], v[part], [m])
                blocks, offsets = self._places(stream, self.length[stream] - m, m)
                self.scores[blocks, :, offsets] = 0.0
                outs.append(fd.window_attention(
                    rot, self.k, self.v, self._table([stream]), self._tensor([self.length[stream]], torch.int32),
                    window=self.budget, sinks=self.sinks, query_start_loc=self._tensor([0, m], torch.int32),
                    max_query_len=m))
                step += m
        if self.length[stream] >= self.budget + self.slack:  # the first decoded token would rank zeros
            self.evict([stream], newest)
        return torch.cat(outs)

    def decode(self, streams, q, k, v):
        """One token of each stream; streams past budget + slack are cut first."""
        full = [s for s in streams if self.length[s] >= self.budget + self.slack]
        for s in full:
            self.evict([s])
        rot = self.append(streams, q, k, v, [1] * len(streams))
        lens = self._tensor([self.length[s] for s in streams], torch.int32)
        return fd.scored_decode(rot, self.k, self.v, self.scores, self._table(streams), lens)

    def evict(self, streams, recent=None):
        """Keep the budget's worth of each stream in fresh pages, the last
        `recent` tokens (the layer's own number if None) among it."""
        recent = self.recent if recent is None else recent
        kept = -(-self.budget // self.block_size)
        new = [[self.free.pop() for _ in range(kept)] for _ in streams]
        lens = self._tensor([self.length[s] for s in streams], torch.int32)
        fd.evict_tokens(self.k, self.v, self.scores, self._table(streams), lens, self._tensor(new, torch.int32),
                        budget=self.budget, sinks=self.sinks, recent=recent)
        for s, pages in zip(streams, new):
            self.free += self.pages[s]
            self.pages[s] = pages
            self.evicted += self.length[s] - self.budget
            self.length[s] = min(self.length[s], self.budget)


def run(streams=4, prompt=3000, tokens=200, seed=0, **layer_options):
    """Serve `streams` prompts and `tokens` decoded tokens; returns the layer
    and the last outputs."""
    layer = BoundedLayer(streams, **layer_options)
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def drawn(n, heads):
        x = torch.randn((n, heads, layer.head_dim), generator=gen, device="cuda")
        return x.to(layer.k.dtype)

    for s in range(streams):
        layer.prompt(s, drawn(prompt, layer.q_heads), drawn(prompt, layer.kv_heads), drawn(prompt, layer.kv_heads))
    out = None
    for _ in range(tokens):
        out = layer.decode(list(range(streams)), drawn(streams, layer.q_heads), drawn(streams, layer.kv_heads),
                           drawn(streams, layer.kv_heads))
    return layer, out


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--streams", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=3000)
    ap.add_argument("--tokens", type=int, default=200)
    ap.add_argument("--budget", type=int, default=2048)
    a = ap.parse_args()
    layer, _ = run(a.streams, a.prompt, a.tokens, budget=a.budget)
    torch.cuda.synchronize()
    print(f"{a.streams} streams of {a.prompt + a.tokens} tokens in {layer.blocks} pages of {layer.block_size}; "
          f"cached now: {layer.length}, evicted: {layer.evicted}, status {fd.device_status()}")


if __name__ == "__main__":
    main()
