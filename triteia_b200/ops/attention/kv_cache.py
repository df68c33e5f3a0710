"""A paged cache of keys and values: [pages, page_size, kv_heads, head_size], in the model's type or as e4m3 codes with one
exponent byte b per token and head (value = code * 2^(b - 127); 127 for a head of zeros, also in a cache that is filled by other
means: paged_attention knows such heads by it).  A token's slot is page * page_size + place."""
import torch

from ..._lib import binding


def new_cache(num_pages, page_size, kv_heads, head_size, dtype=torch.float16, quantised=False, device="cuda"):
    """(key_cache, value_cache, key_exponents, value_exponents); the exponents are None for a cache of `dtype`."""
    shape = (num_pages, page_size, kv_heads, head_size)
    if not quantised:
        return torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device), None, None
    return (torch.zeros(shape, dtype=torch.float8_e4m3fn, device=device), torch.zeros(shape, dtype=torch.float8_e4m3fn, device=device),
            torch.full(shape[:3], 127, dtype=torch.uint8, device=device), torch.full(shape[:3], 127, dtype=torch.uint8, device=device))


def cache_write(key, value, key_cache, value_cache, slots, key_exponents=None, value_exponents=None):
    """Stores key and value [T, kv_heads, head_size] (rows may be parts of a fused projection) at `slots` [T].  A slot outside
    the cache (-1: padding) is skipped; a slot comes at most once in a call."""
    binding.cache_write(key, value, key_cache, value_cache, slots, key_exponents, value_exponents)


def cache_read(key_cache, value_cache, slots, key_exponents=None, value_exponents=None, dtype=None):
    """(key, value) [T, kv_heads, head_size] of the tokens at `slots` as numbers of `dtype` (the cache's own, or for an e4m3
    cache float16 or bfloat16); zeros for a slot outside the cache."""
    return binding.cache_read(key_cache, value_cache, slots, key_exponents, value_exponents, dtype)
