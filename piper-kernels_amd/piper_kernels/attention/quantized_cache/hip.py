"""The cache operators' torch ops: definitions, fakes and where their GPU kernels come from.

``piper_kernels::cache_write``, ``cache_read``, ``cache_attention`` and ``cache_select`` are defined here; their GPU
kernels are native (``csrc/torch_cache.cpp`` over ``include/piper_cache.h``), registered when
``_hip.library.load_torch_kernels`` runs.  The definitions' own body runs only before that, where a process's first call
comes from a compiled graph or the op itself: it registers the kernels and goes there.
"""

from __future__ import annotations

import torch

from ..._hip import library as native

_CACHE = "Tensor cache_key, Tensor cache_key_scale, Tensor cache_value, Tensor cache_value_scale"
_ROWS = "Tensor page_table, Tensor starts, Tensor? counts"
_SCHEMAS = {
    "cache_write": "(Tensor key, Tensor value, Tensor(a!) cache_key, Tensor(b!) cache_key_scale, Tensor(c!) cache_value, "
    f"Tensor(d!) cache_value_scale, Tensor(e!) cache_bounds, Tensor(f!) cache_bound_scale, {_ROWS}) -> ()",
    "cache_read": f"({_CACHE}, {_ROWS}, int size, ScalarType dtype) -> (Tensor, Tensor)",
    "cache_attention": f"(Tensor query, {_CACHE}, {_ROWS}, Tensor? mask, Tensor? selected, float scale) -> Tensor",
    "cache_select": f"(Tensor query, Tensor cache_bounds, Tensor cache_bound_scale, {_ROWS}, int budget) -> Tensor",
}

_library = torch.library.Library("piper_kernels", "FRAGMENT")


def _define(name: str) -> None:
    def first_call(*args):
        device = next(a.device for a in args if isinstance(a, torch.Tensor))
        if device.type != "cuda":
            raise NotImplementedError(f"piper_kernels::{name} runs only on AMD gfx950 (MI355X) HIP devices, got {device}")
        native.load_torch_kernels()
        return getattr(torch.ops.piper_kernels, name)(*args)

    _library.define(name + _SCHEMAS[name])
    _library.impl(name, first_call, "CompositeExplicitAutograd")


for _name in _SCHEMAS:
    _define(_name)


@torch.library.register_fake("piper_kernels::cache_write", lib=_library)
def _cache_write_fake(*_args) -> None:
    return None


@torch.library.register_fake("piper_kernels::cache_read", lib=_library)
def _cache_read_fake(cache_key, _key_scale, _value, _value_scale, page_table, _starts, _counts, size, dtype):
    shape = (page_table.shape[0], cache_key.shape[1], size, cache_key.shape[3])
    return cache_key.new_empty(shape, dtype=dtype), cache_key.new_empty(shape, dtype=dtype)


@torch.library.register_fake("piper_kernels::cache_attention", lib=_library)
def _cache_attention_fake(query, *_args):
    return torch.empty_like(query, memory_format=torch.contiguous_format)


@torch.library.register_fake("piper_kernels::cache_select", lib=_library)
def _cache_select_fake(query, cache_bounds, _bound_scale, _page_table, _starts, _counts, budget):
    return query.new_empty((query.shape[0], cache_bounds.shape[1], query.shape[2], budget), dtype=torch.int32)
