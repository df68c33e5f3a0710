"""Attention of new tokens over a paged cache: single tokens, chunks of prompts, whole prompts and mixtures of them in one
call.  Stands for the decode and extend programs of the reference (triteia/triton/decode_attention.py:30-214,
extend_attention.py:39-170) and for its one-sequence wrapper (triteia/python/ops/attention/sdpa.py:25)."""
from ..._lib import binding


def paged_attention(query, key_cache, value_cache, page_table, lengths, query_starts=None, scale=None, causal=True, window=None,
                    key_exponents=None, value_exponents=None, out=None):
    """query [T, heads, head_size] -> out of the same shape.

    Sequence b has lengths[b] tokens in the cache (int32 [B]), token j on page page_table[b, j // page_size] (int32
    [B, width]).  Its new tokens are the last of them and stand in rows query_starts[b] .. query_starts[b + 1] of query
    (int32 [B + 1]; None: one new token per sequence).  A new token at position p sees the positions up to p (causal; all of
    the sequence otherwise), the last `window` of them where a window is given; a row that sees nothing is zero.  heads is a
    multiple of the cache's heads.  Rows of a given out that belong to no sequence are left as they are, those of a new one are
    zero; a negative page counts as masked.  scale: 1 / sqrt(head_size) by default.

    head_size is 64 or 128, and heads begin on 16-byte boundaries (of an e4m3 cache too, where cache_write is content with 8).  Among
    many single tokens or sequences without new ones, a chunk of hundreds is faster in a call of its own; a page table much wider
    than the sequences are long costs small calls some microseconds.

    What lies in the cache at or beyond a sequence's length, or before the window of all its new tokens, is never used.  Keys and
    values of the other tokens are finite numbers: a NaN or an infinity among them may reach every new token of its sequence,
    also those that do not see it."""
    return binding.paged_attention(query, key_cache, value_cache, page_table, lengths, query_starts, scale, causal, window, key_exponents,
                                   value_exponents, out)
