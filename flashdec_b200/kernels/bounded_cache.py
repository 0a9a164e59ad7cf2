"""Attention over a bounded paged cache: streams longer than their cache.

Not in the reference.  Three operators on the same paged K/V cache as
``decode``:

* :func:`window_attention`: one token, a few drafts or a whole prompt chunk
  per sequence, each query seeing a sliding window and the first tokens
  (sinks);
* :func:`scored_decode`: the decode of one token per sequence that also adds
  up, for every cached token, the attention weight it got;
* :func:`evict_tokens`: the cached tokens that got the least weight leave the
  cache; the others move, in order, to new pages.

Everything runs on the current stream, in kernels of
``libflashdec_b200.so``; the checks are done by the C++ host path and raise
``ValueError``.
"""

from __future__ import annotations

from .. import _lib

__all__ = ["window_attention", "scored_decode", "evict_tokens"]


def window_attention(q, k_cache, v_cache, block_tables, seq_lens, *, window, sinks=0,
                     query_start_loc=None, max_query_len=None, sm_scale=None,
                     kv_layout="token_major", out=None):
    """Attention with a sliding window and sink tokens over a paged cache.

    The queries of sequence ``b`` are its last tokens; their K and V are in
    the cache already and ``seq_lens[b]`` counts them.  A query at position
    ``p`` sees key ``j`` iff ``j <= p`` and (``j > p - window`` or ``j <
    sinks``); a window as long as the sequence is plain causal attention.

    - q: [num_tokens, num_q_heads, head_dim], float16 or bfloat16, head_dim 64
      or 128
    - k_cache, v_cache: [num_blocks, num_kv_heads, block_size, head_dim]
      (``dim_major``: [..., head_dim, block_size]), block_size 8, 16 or 32, any
      strides
    - block_tables [num_seqs, max_blocks_per_seq], seq_lens [num_seqs]: int32 or
      int64.  Pages that hold no visible key are not read: their entries may
      be stale.
    - query_start_loc [num_seqs + 1]: sequence b owns rows
      ``query_start_loc[b]:query_start_loc[b + 1]`` of q; None: one row per
      sequence.  With it, ``max_query_len`` (the longest of them) sizes the
      launch.  Rows no sequence owns are not written.
    - return: like q (``out`` if given).  A query without a visible key (more
      queries than cached tokens, an empty sequence) gets zeros.

    Scores, softmax statistics and sums are fp32; the softmax weights are
    rounded to the cache's type for the product with V.
    """
    hp = _lib.load_hostpath()
    return hp.window_attention(q, k_cache, v_cache, block_tables, seq_lens, window, sinks,
                               query_start_loc, max_query_len, sm_scale, kv_layout, out)


def scored_decode(q, k_cache, v_cache, scores, block_tables, seq_lens, *, sm_scale=None,
                  kv_layout="token_major", out=None):
    """``decode`` that also accumulates each cached token's attention weight.

    - q: [num_seqs, num_q_heads, head_dim]; caches, tables and lengths as in
      :func:`window_attention`
    - scores: [num_blocks, num_kv_heads, block_size] float32, updated in
      place: every token of sequence b gets the softmax weights of the query
      heads that share its KV head added.  The newest token's score is set
      instead, so the slots of tokens that enter the cache one at a time
      through here need no clearing.  Every other slot does: of a prompt or of
      drafts, appended several at once, only the last token is ever the
      newest, and the others' slots hold what their pages' former owner left
      (set them to zero when the tokens are appended).  No two sequences may
      share a page.
    - return: like q (``out`` if given); zeros for an empty sequence.
    """
    hp = _lib.load_hostpath()
    return hp.scored_decode(q, k_cache, v_cache, scores, block_tables, seq_lens, sm_scale,
                            kv_layout, out)


def evict_tokens(k_cache, v_cache, scores, block_tables, seq_lens, new_block_tables, *, budget,
                 sinks=0, recent=0, kv_layout="token_major"):
    """Copy the tokens worth keeping, at most ``budget`` per sequence and KV
    head, to new pages.

    A sequence within its budget keeps every token.  A longer one keeps, per
    KV head, its first ``sinks`` tokens, its last ``recent`` and the best
    scored of the others (equal scores: the lower position first; NaN ranks
    above every number), in their order.  K, V and scores of place i of
    sequence b go to slot ``i % block_size`` of page ``new_block_tables[b, i //
    block_size]``, whose rows have room for ``min(budget, max_blocks_per_seq *
    block_size)`` tokens; the source pages stay as they are (they may be shared with
    other sequences), and the caller frees them afterwards.  New pages must be
    distinct and none of them a source page.

    Keys are copied as cached (already rotated), so the kept tokens keep the
    positions they were rotated by.

    Returns ``(kept, new_seq_lens)``: kept [num_seqs, num_kv_heads, budget]
    int32, the old position of each place (-1 past the new length), and
    new_seq_lens = min(seq_lens, budget) in the dtype of ``seq_lens``.
    """
    hp = _lib.load_hostpath()
    return hp.evict_tokens(k_cache, v_cache, scores, block_tables, seq_lens, new_block_tables,
                           budget, sinks, recent, kv_layout)
