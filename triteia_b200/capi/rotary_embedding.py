"""Rotary position embedding, in place; same functions as
triteia/python/capi/rotary_embedding.py:5-38."""
from .. import triteia_cuda


def rotary_embedding(positions, query, key, head_size, cos_sin_cache, is_neox) -> None:
    triteia_cuda.rotary_embedding(positions, query, key, head_size, cos_sin_cache, is_neox)


def batched_rotary_embedding(positions, query, key, head_size, cos_sin_cache, is_neox, rot_dim,
                             cos_sin_cache_offsets) -> None:
    triteia_cuda.batched_rotary_embedding(positions, query, key, head_size, cos_sin_cache, is_neox, rot_dim,
                                          cos_sin_cache_offsets)


def qk_norm_rotary_embedding(positions, query, key, head_size, cos_sin_cache, is_neox, query_weight=None, key_weight=None,
                             eps=1e-6, query_out=None, key_out=None) -> None:
    """The norm of every query and key head (eps=None: none) and the rotation in one pass, on rows that may be column ranges of a
    fused projection; in place, or into query_out / key_out.  No counterpart in the reference."""
    triteia_cuda.qk_norm_rotary_embedding(positions, query, key, head_size, cos_sin_cache, is_neox, query_weight, key_weight, eps,
                                          query_out, key_out)
