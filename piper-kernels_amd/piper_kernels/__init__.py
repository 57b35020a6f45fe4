"""MI355X-native Piper Attention and SageAttention2++ forward (gfx950 HIP kernels behind a C ABI).

Drop-in for the public operators of jumbledpoophj/piper-kernels
(``src/piper_kernels/__init__.py:3-6``): ``from piper_kernels import piper_attention,
sage_attention_2pp``.  Beside them, without a counterpart there: a paged KV cache in 8 bits and the
attention that reads it (``QuantizedCache``, ``cache_write``, ``cache_read``, ``cache_attention``,
``cache_select``).
"""

from .attention.piper_attention import piper_attention
from .attention.quantized_cache import QuantizedCache, cache_attention, cache_read, cache_select, cache_write
from .attention.sage_attention_2pp import sage_attention_2pp

__all__ = [
    "QuantizedCache",
    "cache_attention",
    "cache_read",
    "cache_select",
    "cache_write",
    "piper_attention",
    "sage_attention_2pp",
]
