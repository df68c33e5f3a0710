"""delta_attention — the attention block of a decoder layer that serves many fine-tuned models at once: the fused q/k/v and
the output projection are a base weight plus the packed delta that each token's index selects; between them stand the norm and
rotation of the heads, the paged cache and the attention over it.  The reference has the two projections
(triteia/python/ops/matmul/sbmm.py:89) and leaves what is between them to the serving engine."""
import torch
import torch.nn as nn

from ..capi import qk_norm_rotary_embedding
from ..ops import cache_write, paged_attention, sbmm_4bit_2_4_native


class delta_attention(nn.Module):
    """Buffers, to be filled by the caller: `qkv_weight` [(heads + 2 kv_heads) * head_size, hidden] and `o_weight` [hidden,
    heads * head_size] fp16, the base model's; per projection the stacked deltas `*_qweight`, `*_meta`, `*_scale` as
    sbmm_4bit_2_4_native takes them; `cos_sin_cache` [max_position, rot_dim] float32; `query_norm` and `key_norm` [head_size]
    with qk_norm."""

    def __init__(self, hidden, heads, kv_heads, head_size, num_deltas, max_position, rot_dim=None, groupsize=-1, qk_norm=False,
                 eps=1e-6, is_neox=True, window=None):
        super().__init__()
        if heads % kv_heads != 0:
            raise ValueError(f"{heads} query heads do not divide into {kv_heads} key heads")
        self.heads, self.kv_heads, self.head_size = heads, kv_heads, head_size
        self.eps, self.is_neox, self.window, self.qk_norm = eps, is_neox, window, qk_norm
        half = dict(dtype=torch.float16)
        for name, k, n in (("qkv", hidden, (heads + 2 * kv_heads) * head_size), ("o", heads * head_size, hidden)):
            self.register_buffer(f"{name}_weight", torch.empty((n, k), **half))
            self.register_buffer(f"{name}_qweight", torch.empty((num_deltas, k // 32, 2 * n), dtype=torch.int32))
            self.register_buffer(f"{name}_meta", torch.empty((num_deltas, n, k // 16), dtype=torch.int16))
            self.register_buffer(f"{name}_scale", torch.empty((num_deltas, 1 if groupsize == -1 else k // groupsize, n), **half))
        self.register_buffer("cos_sin_cache", torch.empty((max_position, head_size if rot_dim is None else rot_dim), dtype=torch.float32))
        self.register_buffer("query_norm", torch.ones(head_size, **half) if qk_norm else None)
        self.register_buffer("key_norm", torch.ones(head_size, **half) if qk_norm else None)

    def forward(self, x, indices, positions, slots, cache, page_table, lengths, query_starts=None):
        """x [T, hidden] fp16, the new tokens of the batch's sequences one after the other; indices [T] delta ids (-1: base model);
        positions int64 [T]; slots int64 [T], where their keys and values go; cache: what new_cache returned; page_table,
        lengths (the new tokens included) and query_starts as paged_attention takes them.  Rows of x behind the last sequence are
        padding (slot -1, position -1): their rows of the output projection's input are zero."""
        q_end = self.heads * self.head_size
        k_end = q_end + self.kv_heads * self.head_size
        qkv = sbmm_4bit_2_4_native(self.qkv_qweight, x, self.qkv_meta, self.qkv_scale, indices, base_weight=self.qkv_weight)
        query, key = qkv[:, :q_end], qkv[:, q_end:k_end]
        qk_norm_rotary_embedding(positions, query, key, self.head_size, self.cos_sin_cache, self.is_neox, self.query_norm, self.key_norm,
                                 self.eps if self.qk_norm else None)
        key_cache, value_cache, key_exponents, value_exponents = cache
        heads = (-1, self.head_size)
        cache_write(key.unflatten(1, heads), qkv[:, k_end:].unflatten(1, heads), key_cache, value_cache, slots, key_exponents, value_exponents)
        out = paged_attention(query.unflatten(1, heads), key_cache, value_cache, page_table, lengths, query_starts, window=self.window,
                              key_exponents=key_exponents, value_exponents=value_exponents)
        return sbmm_4bit_2_4_native(self.o_qweight, out.flatten(1), self.o_meta, self.o_scale, indices, base_weight=self.o_weight)
