"""The quantised paged KV cache and the attention that reads it on MI355X."""

from .dispatch import QuantizedCache, cache_attention, cache_read, cache_select, cache_write

__all__ = ["QuantizedCache", "cache_attention", "cache_read", "cache_select", "cache_write"]
