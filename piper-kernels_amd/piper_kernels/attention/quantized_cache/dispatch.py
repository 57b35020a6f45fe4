"""Public entry points of the quantised paged KV cache on MI355X.

No counterpart in the reference, whose operators quantise K and V inside each call and keep nothing.  The cache keeps
them in 8 bits between calls, as a program that generates needs them: :func:`cache_write` quantises new tokens into
pages, :func:`cache_attention` attends to them (single tokens, drafted trees, chunks of a prompt, selected pages),
:func:`cache_select` selects pages by a bound of their scores, :func:`cache_read` gives K and V back in 16 bits, for
example for ``piper_attention``.

All calls share one way to say where tokens stand.  ``page_table`` (int32 ``[batch, n]``) names the cache page of each 64
positions of a sequence; row ``i < counts[b]`` of a call is position ``starts[b] + i`` (both int32 ``[batch]``;
``counts=None``: every row).  Rows beyond a count are padding: not written, zero in outputs.  All three are read on the GPU
when the kernels run, so a captured graph follows their contents.  Entries outside the cache and positions beyond the table
name no page: nothing is written there and nothing there is seen.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from ..._hip.library import load_library, load_torch_kernels
from ..._hip.targets import AcceleratorTarget
from . import hip  # noqa: F401  (defines the ops)

PAGE = 64  # tokens of a page: the operators' key tile
_DTYPES = (torch.float16, torch.bfloat16)
_CODE_DTYPES = (torch.int8, torch.float8_e4m3fn)
_HEAD_DIMS = (64, 128)
_ops = torch.ops.piper_kernels
_write, _read = _ops.cache_write.default, _ops.cache_read.default
_attention, _select = _ops.cache_attention.default, _ops.cache_select.default


class QuantizedCache(NamedTuple):
    """K and V of ``P`` pages of 64 tokens and ``H`` heads in 8 bits, with an FP32 scale per token and head.

    A row of ``head_dim`` values is held as ``code = round(x * (L / a))`` and ``scale = a / L`` with ``a`` its largest
    magnitude; ``L`` is 127 for INT8 and 448 for FP8 E4M3.  ``bounds`` holds, for full pages, INT8 codes of the largest
    and the smallest key value per feature, which :func:`cache_select` reads.
    """

    key: torch.Tensor  # int8 or float8_e4m3fn [P, H, 64, D]
    key_scale: torch.Tensor  # float32 [P, H, 64]
    value: torch.Tensor  # as key, [P, H, 8, D, 8]: token 8a + j, feature d at [a, d, j]
    value_scale: torch.Tensor  # float32 [P, H, 64]
    bounds: torch.Tensor  # int8 [P, H, 2, D]: largest, smallest
    bound_scale: torch.Tensor  # float32 [P, H]

    @classmethod
    def allocate(
        cls, pages: int, kv_heads: int, head_dim: int, *, dtype: torch.dtype = torch.int8, device: torch.device | str | None = None
    ) -> "QuantizedCache":
        """An empty cache of ``pages`` pages of 64 tokens (codes ``torch.int8`` or ``torch.float8_e4m3fn``)."""
        if pages <= 0 or kv_heads <= 0:
            raise ValueError(f"QuantizedCache needs at least one page and one head, got {pages} and {kv_heads}")
        if head_dim not in _HEAD_DIMS:
            raise ValueError(f"QuantizedCache supports head dimensions 64 and 128, got {head_dim}")
        if dtype not in _CODE_DTYPES:
            raise ValueError(f"QuantizedCache codes must use int8 or float8_e4m3fn, got {dtype}")

        def zeros(*shape: int, dtype: torch.dtype = torch.float32) -> torch.Tensor:
            return torch.zeros(shape, dtype=dtype, device=device)

        return cls(
            zeros(pages, kv_heads, PAGE, head_dim, dtype=torch.int8).view(dtype),
            zeros(pages, kv_heads, PAGE),
            zeros(pages, kv_heads, 8, head_dim, 8, dtype=torch.int8).view(dtype),
            zeros(pages, kv_heads, PAGE),
            zeros(pages, kv_heads, 2, head_dim, dtype=torch.int8),
            zeros(pages, kv_heads),
        )


def _check_cache(operator: str, cache: QuantizedCache) -> tuple[int, int, int, torch.device]:
    """Pages, heads, head size and device of a cache whose arrays belong together."""
    key, key_scale, value, value_scale, bounds, bound_scale = cache
    if key.ndim != 4 or key.shape[2] != PAGE:
        raise ValueError(f"{operator} cache.key must have shape [pages, kv_heads, 64, head_dim], got {tuple(key.shape)}")
    p, h, _, d = key.shape
    device = key.device
    if d not in _HEAD_DIMS:
        raise ValueError(f"{operator} supports head dimensions 64 and 128, got {d}")
    if p == 0 or h == 0:
        raise ValueError(f"{operator} does not accept an empty cache")
    if key.dtype not in _CODE_DTYPES:
        raise ValueError(f"{operator} cache.key must use int8 or float8_e4m3fn, got {key.dtype}")
    for name, tensor, shape, dtype in (
        ("key", key, key.shape, key.dtype),
        ("key_scale", key_scale, (p, h, PAGE), torch.float32),
        ("value", value, (p, h, 8, d, 8), key.dtype),
        ("value_scale", value_scale, (p, h, PAGE), torch.float32),
        ("bounds", bounds, (p, h, 2, d), torch.int8),
        ("bound_scale", bound_scale, (p, h), torch.float32),
    ):
        if tensor.shape != shape or tensor.dtype is not dtype:
            raise ValueError(
                f"{operator} cache.{name} must be {dtype} of shape {tuple(shape)}, got {tensor.dtype} {tuple(tensor.shape)}"
            )
        if not tensor.is_contiguous():
            raise ValueError(f"{operator} cache.{name} must be contiguous")
        if tensor.device != device:
            raise ValueError(f"{operator} cache.{name} must be on {device} as cache.key is, got {tensor.device}")
    return p, h, d, device


def _check_rows(
    operator: str, page_table: torch.Tensor, starts: torch.Tensor, counts: torch.Tensor | None, batch: int, device: torch.device
) -> None:
    for name, tensor, ndim in (("page_table", page_table, 2), ("starts", starts, 1), ("counts", counts, 1)):
        if tensor is None and name == "counts":
            continue
        if tensor.ndim != ndim or tensor.shape[0] != batch or tensor.shape[-1] == 0 or tensor.dtype is not torch.int32:
            raise ValueError(
                f"{operator} {name} must be an int32 tensor of shape {'[batch, pages]' if ndim == 2 else '[batch]'} with batch {batch}, "
                f"got {tensor.dtype} {tuple(tensor.shape)}"
            )
        if tensor.stride(-1) != 1 and tensor.shape[-1] != 1:
            raise ValueError(f"{operator} {name}'s last dimension must be contiguous")
        if tensor.device != device:
            raise ValueError(f"{operator} {name} must be on {device} as the cache is, got {tensor.device}")


def _check_tokens(operator: str, name: str, tensor: torch.Tensor, head_dim: int, device: torch.device) -> None:
    if tensor.ndim != 4:
        raise ValueError(f"{operator} {name} must have shape [batch, heads, tokens, head_dim], got {tuple(tensor.shape)}")
    if tensor.dtype not in _DTYPES:
        raise ValueError(f"{operator} {name} must use float16 or bfloat16, got {tensor.dtype}")
    if tensor.layout is not torch.strided:
        raise ValueError(f"{operator} {name} must use strided layout")
    if tensor.shape[3] != head_dim:
        raise ValueError(f"{operator} {name} must have the cache's head dimension {head_dim}, got {tensor.shape[3]}")
    if tensor.stride(-1) != 1:
        raise ValueError(f"{operator} {name}'s head dimension must be contiguous")
    if tensor.shape[0] == 0 or tensor.shape[1] == 0 or tensor.shape[2] == 0:
        raise ValueError(f"{operator} does not accept an empty {name}, got {tuple(tensor.shape)}")
    if tensor.device != device:
        raise ValueError(f"{operator} {name} must be on {device} as the cache is, got {tensor.device}")
    _check_grad(operator, tensor)


def _check_grad(operator: str, tensor: torch.Tensor) -> None:
    if tensor.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{operator} is an inference-only operator and does not support autograd")


def _check_query(operator: str, query: torch.Tensor, kv_heads: int, head_dim: int, device: torch.device) -> None:
    _check_tokens(operator, "query", query, head_dim, device)
    if query.shape[1] % kv_heads != 0:
        raise ValueError(f"{operator} query heads must be a multiple of the cache's {kv_heads}, got {query.shape[1]}")


def _require_device(operator: str, device: torch.device) -> None:
    target = AcceleratorTarget.from_device(device)
    if not target.supports_piper_mi355x:
        raise NotImplementedError(
            f"{operator} runs only on AMD gfx950 (MI355X) HIP devices; "
            f"got backend={target.backend!r} architecture={target.architecture!r}"
        )
    if not torch.compiler.is_compiling():
        load_library()  # raises LibraryUnavailableError (a RuntimeError) if the library is missing
        load_torch_kernels()
        _ready.add(device)


_ready: set[torch.device] = set()  # gfx950 devices, once the kernels are loaded


def _call(op, args: tuple, device: torch.device, check):
    """``op(*args)``.  ``check()`` raises what is wrong with a call.  The op's GPU kernel checks everything before it
    launches anything, so where that is known to run, the words are looked for only after a refusal."""
    if torch.compiler.is_compiling() or device not in _ready:
        check()
        return op(*args)
    try:
        return op(*args)
    except Exception:
        check()
        raise


def cache_write(
    cache: QuantizedCache,
    key: torch.Tensor,
    value: torch.Tensor,
    page_table: torch.Tensor,
    starts: torch.Tensor,
    counts: torch.Tensor | None = None,
) -> None:
    """Quantise new tokens' keys and values into the cache, in place.

    ``key`` and ``value`` are ``[batch, kv_heads, tokens, head_dim]`` in FP16 or BF16.  Every page whose last slot is
    among the written ones also gets its bounds, from all 64 keys that it then holds; the bounds of other pages are
    left, and :func:`cache_select` does not read them, since a sequence's last page is always selected.  Writing positions
    again (after drafted tokens were rejected) is ordinary use.  Within one call two rows must not name the same slot, nor
    two sequences a page that either fills.  A token with an infinity or a NaN makes NaN of the rows that attend to it
    and of nothing else.
    """
    operator = "cache_write"

    def check() -> None:
        _, h, d, device = _check_cache(operator, cache)
        _check_tokens(operator, "key", key, d, device)
        _check_tokens(operator, "value", value, d, device)
        if key.shape != value.shape or key.dtype is not value.dtype:
            raise ValueError(
                f"{operator} key and value must share shape and dtype, got {key.dtype} {tuple(key.shape)} and {value.dtype} {tuple(value.shape)}"
            )
        if key.shape[1] != h:
            raise ValueError(f"{operator} key and value must have the cache's {h} heads, got {key.shape[1]}")
        _check_rows(operator, page_table, starts, counts, key.shape[0], device)
        _require_device(operator, device)

    _check_grad(operator, key)
    _check_grad(operator, value)
    _call(_write, (key, value, *cache, page_table, starts, counts), key.device, check)


def cache_read(
    cache: QuantizedCache,
    page_table: torch.Tensor,
    starts: torch.Tensor,
    counts: torch.Tensor | None = None,
    *,
    size: int,
    dtype: torch.dtype = torch.bfloat16,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of positions ``starts[b] + i`` as ``[batch, kv_heads, size, head_dim]`` in ``dtype`` (FP16 or BF16):
    the values that the codes stand for, rounded once; zero where ``i >= counts[b]`` or the table names no page."""
    operator = "cache_read"

    def check() -> None:
        _, _, _, device = _check_cache(operator, cache)
        if dtype not in _DTYPES:
            raise ValueError(f"{operator} dtype must be float16 or bfloat16, got {dtype}")
        if size <= 0:
            raise ValueError(f"{operator} size must be positive, got {size}")
        if page_table.ndim != 2 or page_table.shape[0] == 0:
            raise ValueError(f"{operator} page_table must be an int32 tensor of shape [batch, pages], got {tuple(page_table.shape)}")
        _check_rows(operator, page_table, starts, counts, page_table.shape[0], device)
        _require_device(operator, device)

    return _call(_read, (*cache[:4], page_table, starts, counts, size, dtype), page_table.device, check)


def cache_attention(
    query: torch.Tensor,
    cache: QuantizedCache,
    page_table: torch.Tensor,
    starts: torch.Tensor,
    counts: torch.Tensor | None = None,
    *,
    mask: torch.Tensor | None = None,
    selected: torch.Tensor | None = None,
    scale: float | None = None,
) -> torch.Tensor:
    """Attention of new tokens over the cache, which holds their own keys and values too (:func:`cache_write` first).

    ``query`` is ``[batch, heads, tokens, head_dim]`` in FP16 or BF16; ``heads`` is a multiple of the cache's, and query head
    ``h`` reads K/V head ``h // (heads // kv_heads)``.  ``scale`` defaults to ``head_dim**-0.5``.  What row ``i`` of a
    sequence sees:

    * by default positions ``0 .. starts[b] + i``: one token of a step, or a chunk of a prompt;
    * with ``mask`` (bool ``[batch or 1, tokens, tokens]``), positions before ``starts[b]`` and the new tokens ``j`` with
      ``mask[b, i, j]`` and ``j < counts[b]``: a tree of drafted tokens, each of which sees itself and its ancestors;
    * with ``selected`` (int32 ``[batch, kv_heads, tokens, budget]``, what :func:`cache_select` returns), positions
      ``0 .. starts[b] + i`` in those of the sequence's pages.  Negative entries and such beyond the table name no page; a
      page named twice counts twice.

    Scores, softmax statistics and sums are FP32.  Rows that see nothing are zero.  Inference only.
    """
    operator = "cache_attention"

    def check() -> None:
        _, h, d, device = _check_cache(operator, cache)
        _check_query(operator, query, h, d, device)
        batch, _, tokens, _ = query.shape
        _check_rows(operator, page_table, starts, counts, batch, device)
        if mask is not None:
            if selected is not None:
                raise ValueError(f"{operator} takes a mask or selected pages, not both")
            if mask.dtype is not torch.bool or mask.ndim != 3 or mask.shape[0] not in (1, batch) or mask.shape[1:] != (tokens, tokens):
                raise ValueError(
                    f"{operator} mask must be a bool tensor of shape [{batch} or 1, {tokens}, {tokens}], got {mask.dtype} {tuple(mask.shape)}"
                )
            if mask.device != device:
                raise ValueError(f"{operator} mask must be on {device} as the cache is, got {mask.device}")
        if selected is not None:
            if selected.dtype is not torch.int32 or selected.ndim != 4 or selected.shape[:3] != (batch, h, tokens) or selected.shape[3] == 0:
                raise ValueError(
                    f"{operator} selected must be an int32 tensor of shape [{batch}, {h}, {tokens}, budget], "
                    f"got {selected.dtype} {tuple(selected.shape)}"
                )
            if selected.device != device:
                raise ValueError(f"{operator} selected must be on {device} as the cache is, got {selected.device}")
        if not math.isfinite(converted) or converted <= 0:
            raise ValueError(f"{operator} scale must be finite and positive, got {scale}")
        _require_device(operator, device)

    _check_grad(operator, query)
    converted = float(scale) if scale is not None else query.shape[3] ** -0.5 if query.ndim == 4 and query.shape[3] else 1.0
    return _call(_attention, (query, *cache[:4], page_table, starts, counts, mask, selected, converted), query.device, check)


def cache_select(
    query: torch.Tensor,
    cache: QuantizedCache,
    page_table: torch.Tensor,
    starts: torch.Tensor,
    counts: torch.Tensor | None = None,
    *,
    budget: int,
) -> torch.Tensor:
    """The ``budget`` pages that each new token attends to, per K/V head: int32 ``[batch, kv_heads, tokens, budget]`` of page
    numbers within the sequence, ascending, then -1.

    The page of the token's own position is always among them; the others are the pages before it (all full) whose bounds
    allow the largest scores, ties to the lower page.  A page's score is the largest over the K/V head's query heads of
    ``s * sum_d (max(c[d], 0) * upper[d] + min(c[d], 0) * lower[d])``, times the bounds' scale, with the query row held as INT8 codes ``c``
    and scale ``s`` as the cache holds rows: the sum is one of integers, so the selection does not depend on the order of
    evaluation.
    """
    operator = "cache_select"

    def check() -> None:
        _, h, d, device = _check_cache(operator, cache)
        _check_query(operator, query, h, d, device)
        _check_rows(operator, page_table, starts, counts, query.shape[0], device)
        if budget <= 0:
            raise ValueError(f"{operator} budget must be positive, got {budget}")
        _require_device(operator, device)

    _check_grad(operator, query)
    return _call(_select, (query, cache.bounds, cache.bound_scale, page_table, starts, counts, budget), query.device, check)
