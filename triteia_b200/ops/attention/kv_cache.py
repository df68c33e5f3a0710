"""A paged cache of keys and values: [pages, page_size, kv_heads, head_size], in the model's type or as e4m3 codes with one
exponent byte b per token and head (value = code * 2^(b - 127)).  A token's slot is page * page_size + place."""
import torch

from ... import _lib
from ..._lib import lib, ptr, stream_of, dev_of


def new_cache(num_pages, page_size, kv_heads, head_size, dtype=torch.float16, quantised=False, device="cuda"):
    """(key_cache, value_cache, key_exponents, value_exponents); the exponents are None for a cache of `dtype`."""
    shape = (num_pages, page_size, kv_heads, head_size)
    if not quantised:
        return torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device), None, None
    return (torch.zeros(shape, dtype=torch.float8_e4m3fn, device=device), torch.zeros(shape, dtype=torch.float8_e4m3fn, device=device),
            torch.full(shape[:3], 127, dtype=torch.uint8, device=device), torch.full(shape[:3], 127, dtype=torch.uint8, device=device))


def check_cache(key_cache, value_cache, key_exponents, value_exponents, dtype, device):
    """(pages, page size, heads, head size, the six strides) of a cache that holds `dtype` or e4m3 with exponents."""
    if key_cache.dim() != 4 or key_cache.shape != value_cache.shape or key_cache.stride() != value_cache.stride():
        raise RuntimeError("key_cache and value_cache must be [pages, page_size, kv_heads, head_size] with the same strides")
    pages, page_size, heads, size = key_cache.shape
    s = key_cache.stride()
    if s[3] != 1 or page_size == 0 or heads == 0:
        raise RuntimeError("a cache needs a page size, heads and a contiguous last dimension")
    want = dtype if key_exponents is None else torch.float8_e4m3fn
    if key_cache.dtype != want or value_cache.dtype != want:
        raise RuntimeError(f"the cache holds {key_cache.dtype} and {value_cache.dtype}: {want} is needed "
                           f"{'without' if key_exponents is None else 'with'} exponents")
    if (key_exponents is None) != (value_exponents is None):
        raise RuntimeError("key_exponents and value_exponents go together")
    if key_cache.device != device or value_cache.device != device:
        raise RuntimeError(f"the cache must be on {device}")
    if key_exponents is None:
        return pages, page_size, heads, size, s[0], s[1], s[2], 0, 0, 0
    for e in (key_exponents, value_exponents):
        if e.dtype != torch.uint8 or e.shape != key_cache.shape[:3] or e.stride() != key_exponents.stride() or e.device != device:
            raise RuntimeError("exponents must be uint8 [pages, page_size, kv_heads] on the cache's device, both with the same strides")
    es = key_exponents.stride()
    return pages, page_size, heads, size, s[0], s[1], s[2], es[0], es[1], es[2]


def _check_slots(slots, n, device):
    if slots.dtype != torch.int64 or slots.dim() != 1 or not slots.is_contiguous() or slots.device != device:
        raise RuntimeError(f"slots must be a contiguous one-dimensional int64 tensor on {device}")
    if n is not None and slots.size(0) != n:
        raise RuntimeError(f"{slots.size(0)} slots for {n} tokens")


def cache_write(key, value, key_cache, value_cache, slots, key_exponents=None, value_exponents=None):
    """Stores key and value [T, kv_heads, head_size] (rows may be parts of a fused projection) at `slots` [T].  A slot outside
    the cache (-1: padding) is skipped; a slot comes at most once in a call."""
    dev = dev_of(key)
    if key.dim() != 3 or key.shape != value.shape or key.dtype != value.dtype or value.device != key.device:
        raise RuntimeError("key and value must be [tokens, kv_heads, head_size] of one dtype on one device")
    if key.stride(2) != 1 or value.stride(2) != 1:
        raise RuntimeError("key and value need a contiguous last dimension")
    pages, page_size, heads, size, *strides = check_cache(key_cache, value_cache, key_exponents, value_exponents, key.dtype, key.device)
    T = key.size(0)
    if key.size(1) != heads or key.size(2) != size:
        raise RuntimeError(f"key of shape {tuple(key.shape)}: the cache needs [{T}, {heads}, {size}]")
    _check_slots(slots, T, key.device)
    err = lib.trb_cache_write(ptr(key), ptr(value), ptr(slots), ptr(key_cache), ptr(value_cache), ptr(key_exponents),
                              ptr(value_exponents), T, heads, size, page_size, pages, key.stride(0), key.stride(1), value.stride(0),
                              value.stride(1), *strides, _lib.dtype_tag(key.dtype), dev, stream_of(key))
    if err == _lib.ERR_PROB_SHAPE:
        raise RuntimeError(f"No suitable kernel. head_size={size} (a multiple of 8 up to 256, heads on 16-byte boundaries)")
    _lib.check(err, "cache_write")


def cache_read(key_cache, value_cache, slots, key_exponents=None, value_exponents=None, dtype=None):
    """(key, value) [T, kv_heads, head_size] of the tokens at `slots` as numbers of `dtype` (the cache's own, or for an e4m3
    cache float16 or bfloat16); zeros for a slot outside the cache."""
    dev = dev_of(key_cache)
    if dtype is None:
        dtype = key_cache.dtype
    tag = _lib.dtype_tag(dtype)
    pages, page_size, heads, size, *strides = check_cache(key_cache, value_cache, key_exponents, value_exponents, dtype, key_cache.device)
    _check_slots(slots, None, key_cache.device)
    T = slots.size(0)
    key = torch.empty(T, heads, size, dtype=dtype, device=key_cache.device)
    value = torch.empty_like(key)
    err = lib.trb_cache_read(ptr(key_cache), ptr(value_cache), ptr(key_exponents), ptr(value_exponents), ptr(slots), ptr(key),
                             ptr(value), T, heads, size, page_size, pages, *strides, tag, dev, stream_of(key_cache))
    if err == _lib.ERR_PROB_SHAPE:
        raise RuntimeError(f"No suitable kernel. head_size={size} (a multiple of 8 up to 256, heads on 16-byte boundaries)")
    _lib.check(err, "cache_read")
    return key, value
