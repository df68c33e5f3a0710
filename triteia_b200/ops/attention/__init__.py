"""What stands between a layer's q/k/v projection and its output projection: the paged cache and the attention over it.
The reference keeps attention next to its operators too (triteia/python/ops/attention/, triteia/triton/)."""
from .kv_cache import cache_read, cache_write, new_cache
from .paged import paged_attention
