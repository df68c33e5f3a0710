"""Attention of new tokens over a paged cache: single tokens, chunks of prompts, whole prompts and mixtures of them in one
call.  Stands for the decode and extend programs of the reference (triteia/triton/decode_attention.py:30-214,
extend_attention.py:39-170) and for its one-sequence wrapper (triteia/python/ops/attention/sdpa.py:25)."""
import torch

from ... import _lib
from ..._lib import lib, ptr, stream_of, dev_of
from .kv_cache import check_cache


def paged_attention(query, key_cache, value_cache, page_table, lengths, query_starts=None, scale=None, causal=True, window=None,
                    key_exponents=None, value_exponents=None, out=None):
    """query [T, heads, head_size] -> out of the same shape.

    Sequence b has lengths[b] tokens in the cache (int32 [B]), token j on page page_table[b, j // page_size] (int32
    [B, width]).  Its new tokens are the last of them and stand in rows query_starts[b] .. query_starts[b + 1] of query
    (int32 [B + 1]; None: one new token per sequence).  A new token at position p sees the positions up to p (causal; all of
    the sequence otherwise), the last `window` of them where a window is given; a row that sees nothing is zero.  heads is a
    multiple of the cache's heads.  Rows of out that belong to no sequence are left as they are; a negative page counts as
    masked.  scale: 1 / sqrt(head_size) by default."""
    dev = dev_of(query)
    if query.dim() != 3 or query.stride(2) != 1:
        raise RuntimeError("query must be [tokens, heads, head_size] with a contiguous last dimension")
    T, heads, size = query.shape
    device = query.device
    pages, page_size, kv_heads, kv_size, *strides = check_cache(key_cache, value_cache, key_exponents, value_exponents, query.dtype, device)
    if kv_size != size or heads == 0 or heads % kv_heads != 0:
        raise RuntimeError(f"query heads {heads} x {size} do not go with key heads {kv_heads} x {kv_size}")
    if page_table.dim() != 2 or page_table.dtype != torch.int32 or page_table.device != device or (page_table.size(1) > 1 and page_table.stride(1) != 1):
        raise RuntimeError(f"page_table must be int32 [sequences, pages] with contiguous rows on {device}")
    B = page_table.size(0)
    for t, n, want in ((lengths, "lengths", B), (query_starts, "query_starts", B + 1)):
        if t is not None and (t.dtype != torch.int32 or t.dim() != 1 or t.size(0) != want or not t.is_contiguous() or t.device != device):
            raise RuntimeError(f"{n} must be a contiguous int32 tensor of {want} entries on {device}")
    if query_starts is None and T != B:
        raise RuntimeError(f"{T} tokens for {B} sequences: query_starts is needed")
    if window is not None and (window <= 0 or not causal):
        raise RuntimeError("a window is a positive number of tokens and needs causal=True")
    if out is None:
        out = torch.empty(T, heads, size, dtype=query.dtype, device=device)
    elif out.shape != query.shape or out.dtype != query.dtype or out.device != device or out.stride(2) != 1:
        raise RuntimeError("out must have the shape, dtype and device of query and a contiguous last dimension")
    err = lib.trb_paged_attention(ptr(query), ptr(key_cache), ptr(value_cache), ptr(key_exponents), ptr(value_exponents),
                                  ptr(page_table), ptr(lengths), ptr(query_starts), ptr(out), T, B, heads, kv_heads, size, page_size,
                                  pages, page_table.stride(0), page_table.size(1), query.stride(0), query.stride(1), out.stride(0),
                                  out.stride(1), *strides, float(size ** -0.5 if scale is None else scale), int(causal), window or 0,
                                  _lib.dtype_tag(query.dtype), dev, stream_of(query))
    if err in (_lib.ERR_PROB_SHAPE, _lib.ERR_KERN_SHAPE):
        raise RuntimeError(f"No suitable kernel. head_size={size} dtype={query.dtype} (heads of 64 or 128, rows on 16-byte boundaries)")
    _lib.check(err, "paged_attention")
    return out
