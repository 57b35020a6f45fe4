"""The quantised cache on the CPU: refusals of the public functions and of the C ABI, the header against its bindings,
the index arithmetic that keeps the kernels inside their buffers, and the model the GPU tests compare with."""

from __future__ import annotations

import ctypes
import math
import re
import subprocess
from pathlib import Path

import pytest
import torch

import piper_kernels
from _cache import PAGE, Model, quantise, table_of, tokens_of
from piper_kernels import QuantizedCache, cache_attention, cache_read, cache_select, cache_write
from piper_kernels._hip import library as native

REPO = Path(__file__).resolve().parents[1]
HEADER = REPO / "include" / "piper_cache.h"


def _call(**changes):
    """Arguments of a good call on CPU tensors, with changes."""
    cache = QuantizedCache.allocate(6, 2, 64)
    args = {
        "cache": cache,
        "key": torch.zeros((2, 2, 3, 64), dtype=torch.float16),
        "value": torch.zeros((2, 2, 3, 64), dtype=torch.float16),
        "query": torch.zeros((2, 4, 3, 64), dtype=torch.float16),
        "page_table": torch.zeros((2, 3), dtype=torch.int32),
        "starts": torch.zeros(2, dtype=torch.int32),
        "counts": None,
        "mask": None,
        "selected": None,
        "scale": None,
        "size": 3,
        "dtype": torch.float16,
        "budget": 2,
    }
    replaced = {k: v for k, v in changes.items() if k in cache._fields and k not in ("key", "value")}
    replaced |= {k[len("cache_"):]: v for k, v in changes.items() if k in ("cache_key", "cache_value")}
    args |= {k: v for k, v in changes.items() if k in args}
    args["cache"] = args["cache"]._replace(**replaced)
    return args


def _write(a):
    return cache_write(a["cache"], a["key"], a["value"], a["page_table"], a["starts"], a["counts"])


def _read(a):
    return cache_read(a["cache"], a["page_table"], a["starts"], a["counts"], size=a["size"], dtype=a["dtype"])


def _attention(a):
    return cache_attention(a["query"], a["cache"], a["page_table"], a["starts"], a["counts"], mask=a["mask"], selected=a["selected"],
                           scale=a["scale"])


def _select(a):
    return cache_select(a["query"], a["cache"], a["page_table"], a["starts"], a["counts"], budget=a["budget"])


EVERY = {"write": _write, "read": _read, "attention": _attention, "select": _select}


def test_package_exports_the_cache() -> None:
    for name in ("QuantizedCache", "cache_write", "cache_read", "cache_attention", "cache_select"):
        assert name in piper_kernels.__all__ and hasattr(piper_kernels, name)


@pytest.mark.parametrize("name", EVERY)
def test_a_good_call_is_refused_off_the_gpu_only(name) -> None:
    with pytest.raises(NotImplementedError, match="gfx950"):
        EVERY[name](_call())
    with pytest.raises(NotImplementedError, match="gfx950"):
        a = _call(counts=torch.ones(2, dtype=torch.int32))
        EVERY[name](a)


@pytest.mark.parametrize("name", EVERY)
@pytest.mark.parametrize("change, message", [
    ({"cache_key": torch.zeros((6, 2, 32, 64), dtype=torch.int8)}, r"\[pages, kv_heads, 64, head_dim\]"),
    ({"cache_key": torch.zeros((6, 2, 64, 96), dtype=torch.int8)}, "head dimensions 64 and 128"),
    ({"cache_key": torch.zeros((0, 2, 64, 64), dtype=torch.int8)}, "empty cache"),
    ({"cache_key": torch.zeros((6, 2, 64, 64), dtype=torch.uint8)}, "int8 or float8_e4m3fn"),
    ({"cache_key": torch.zeros((6, 2, 64, 64), dtype=torch.int8).transpose(0, 1).contiguous().transpose(0, 1)}, "key must be contiguous"),
    ({"cache_value": torch.zeros((6, 2, 64, 64), dtype=torch.int8)}, "cache.value must be"),
    ({"cache_value": torch.zeros((6, 2, 8, 64, 8), dtype=torch.int8).view(torch.float8_e4m3fn)}, "cache.value must be"),
    ({"key_scale": torch.zeros((6, 2, 64), dtype=torch.float16)}, "cache.key_scale must be"),
    ({"value_scale": torch.zeros((6, 2, 32))}, "cache.value_scale must be"),
    ({"bounds": torch.zeros((6, 2, 64), dtype=torch.int8)}, "cache.bounds must be"),
    ({"bound_scale": torch.zeros((6, 2, 1))}, "cache.bound_scale must be"),
    ({"key_scale": torch.zeros((6, 2, 64), device="meta")}, "cache.key_scale must be on cpu"),
    ({"page_table": torch.zeros((2, 3), dtype=torch.int64)}, "page_table must be an int32"),
    ({"page_table": torch.zeros((2, 0), dtype=torch.int32)}, "page_table must be an int32"),
    ({"page_table": torch.zeros(2, dtype=torch.int32)}, "page_table must be an int32"),
    ({"page_table": torch.zeros((3, 2), dtype=torch.int32).t()}, "page_table's last dimension"),
    ({"page_table": torch.zeros((2, 3), dtype=torch.int32, device="meta")}, "page_table must be on cpu"),
    ({"starts": torch.zeros(3, dtype=torch.int32)}, "starts must be an int32"),
    ({"starts": torch.zeros(2)}, "starts must be an int32"),
    ({"counts": torch.zeros((2, 1), dtype=torch.int32)}, "counts must be an int32"),
    ({"counts": torch.zeros(4, dtype=torch.int32)[::2]}, "counts's last dimension"),
])
def test_refusals_of_every_call(name, change, message) -> None:
    with pytest.raises(ValueError, match=message):
        EVERY[name](_call(**change))


@pytest.mark.parametrize("name, change, message", [
    ("write", {"key": torch.zeros((2, 2, 64), dtype=torch.float16)}, r"\[batch, heads, tokens, head_dim\]"),
    ("write", {"key": torch.zeros((2, 2, 3, 64))}, "key must use float16 or bfloat16"),
    ("write", {"value": torch.zeros((2, 2, 3, 64), dtype=torch.bfloat16)}, "share shape and dtype"),
    ("write", {"value": torch.zeros((2, 2, 4, 64), dtype=torch.float16)}, "share shape and dtype"),
    ("write", {"key": torch.zeros((2, 2, 3, 128), dtype=torch.float16)}, "cache's head dimension 64"),
    ("write", {"key": torch.zeros((2, 4, 3, 64), dtype=torch.float16), "value": torch.zeros((2, 4, 3, 64), dtype=torch.float16)}, "cache's 2 heads"),
    ("write", {"key": torch.zeros((2, 2, 0, 64), dtype=torch.float16)}, "empty key"),
    ("write", {"key": torch.zeros((2, 2, 3, 128), dtype=torch.float16)[..., ::2]}, "head dimension must be contiguous"),
    ("read", {"size": 0}, "size must be positive"),
    ("read", {"dtype": torch.float32}, "dtype must be float16 or bfloat16"),
    ("read", {"page_table": torch.zeros((0, 3), dtype=torch.int32)}, "page_table must be an int32"),
    ("attention", {"query": torch.zeros((2, 3, 3, 64), dtype=torch.float16)}, "multiple of the cache's 2"),
    ("attention", {"query": torch.zeros((2, 4, 3, 64))}, "query must use float16 or bfloat16"),
    ("attention", {"query": torch.zeros((2, 4, 0, 64), dtype=torch.float16)}, "empty query"),
    ("attention", {"mask": torch.ones((2, 3, 3))}, "mask must be a bool tensor"),
    ("attention", {"mask": torch.ones((3, 3, 3), dtype=torch.bool)}, "mask must be a bool tensor"),
    ("attention", {"mask": torch.ones((2, 3, 4), dtype=torch.bool)}, "mask must be a bool tensor"),
    ("attention", {"mask": torch.ones((2, 3, 3), dtype=torch.bool, device="meta")}, "mask must be on cpu"),
    ("attention", {"selected": torch.zeros((2, 2, 3, 0), dtype=torch.int32)}, "selected must be an int32"),
    ("attention", {"selected": torch.zeros((2, 4, 3, 1), dtype=torch.int32)}, "selected must be an int32"),
    ("attention", {"selected": torch.zeros((2, 2, 3, 1), dtype=torch.int64)}, "selected must be an int32"),
    ("attention", {"mask": torch.ones((2, 3, 3), dtype=torch.bool), "selected": torch.zeros((2, 2, 3, 1), dtype=torch.int32)}, "not both"),
    ("attention", {"scale": 0.0}, "scale must be finite and positive"),
    ("attention", {"scale": math.inf}, "scale must be finite and positive"),
    ("select", {"budget": 0}, "budget must be positive"),
    ("select", {"query": torch.zeros((2, 3, 3, 64), dtype=torch.float16)}, "multiple of the cache's 2"),
])
def test_refusals(name, change, message) -> None:
    with pytest.raises(ValueError, match=message):
        EVERY[name](_call(**change))


@pytest.mark.parametrize("name, tensor", [("write", "key"), ("write", "value"), ("attention", "query"), ("select", "query")])
def test_inference_only(name, tensor) -> None:
    a = _call()
    a[tensor] = a[tensor].clone().requires_grad_()
    with pytest.raises(RuntimeError, match="inference-only"):
        EVERY[name](a)
    with torch.no_grad(), pytest.raises(NotImplementedError):
        EVERY[name](a)


@pytest.mark.parametrize("args, dtype, message", [
    ((0, 2, 64), torch.int8, "at least one page"),
    ((1, 0, 64), torch.int8, "at least one page"),
    ((1, 1, 96), torch.int8, "64 and 128"),
    ((1, 1, 64), torch.uint8, "int8 or float8_e4m3fn"),
])
def test_allocate_refuses(args, dtype, message) -> None:
    with pytest.raises(ValueError, match=message):
        QuantizedCache.allocate(*args, dtype=dtype)


def test_ops_have_fakes() -> None:
    """Shapes and types without a device, as a compiler asks for them."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        a = _call()
        ops, where = torch.ops.piper_kernels, (a["page_table"], a["starts"], None)
        key, value = ops.cache_read(*a["cache"][:4], *where, 7, torch.bfloat16)
        assert key.shape == value.shape == (2, 2, 7, 64) and key.dtype is torch.bfloat16
        out = ops.cache_attention(a["query"].transpose(1, 2).contiguous().transpose(1, 2), *a["cache"][:4], *where, None, None, 1.0)
        assert out.shape == (2, 4, 3, 64) and out.is_contiguous() and out.dtype is torch.float16
        pages = ops.cache_select(a["query"], a["cache"].bounds, a["cache"].bound_scale, *where, 5)
        assert pages.shape == (2, 2, 3, 5) and pages.dtype is torch.int32
        assert ops.cache_write(a["key"], a["value"], *a["cache"], *where) is None
    a = _call()
    with pytest.raises(NotImplementedError, match="gfx950"):
        torch.ops.piper_kernels.cache_write(a["key"], a["value"], *a["cache"], a["page_table"], a["starts"], None)


# ---- C ABI ------------------------------------------------------------------------------------------------------------

STRUCTS = {
    "piper_cache": native.PiperCache,
    "piper_cache_rows": native.PiperCacheRows,
    "piper_cache_write_args": native.PiperCacheWriteArgs,
    "piper_cache_read_args": native.PiperCacheReadArgs,
    "piper_cache_attention_args": native.PiperCacheAttentionArgs,
    "piper_cache_select_args": native.PiperCacheSelectArgs,
}


@pytest.fixture(scope="module")
def lib() -> native.NativeLibrary:
    if not native.library_available():
        pytest.fail("libpiper_mi355x.so is not built; run __graft_entry__.build()")
    return native.load_library()


def test_header_declares_exactly_the_bound_symbols(lib) -> None:
    declared = set(re.findall(r"^\s*int\s+(piper_\w+)\s*\(", HEADER.read_text(), re.MULTILINE))
    assert declared == set(native.CACHE_EXPORTED_SYMBOLS)
    assert all(lib.has_symbol(name) for name in declared)


def test_structures_and_constants_match_the_header(tmp_path) -> None:
    lines = ['#include <stdio.h>', '#include "piper_cache.h"', "int main(void) {"]
    for cname, cls in STRUCTS.items():
        lines.append(f'  printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname}.{f[0]} %zu\\n", offsetof({cname}, {f[0]}));' for f in cls._fields_]
    lines.append('  printf("constants %d%d%d%d\\n", PIPER_CACHE_ABI_VERSION, PIPER_CACHE_PAGE, PIPER_CACHE_INT8, PIPER_CACHE_FP8);')
    lines.append("  return 0; }")
    (tmp_path / "abi.c").write_text("\n".join(lines))
    subprocess.run(["gcc", "-Wall", "-Werror", f"-I{REPO / 'include'}", str(tmp_path / "abi.c"), "-o", str(tmp_path / "abi")], check=True)
    got = dict(line.rsplit(" ", 1) for line in subprocess.run([str(tmp_path / "abi")], capture_output=True, text=True).stdout.splitlines())
    for cname, cls in STRUCTS.items():
        assert int(got[cname]) == ctypes.sizeof(cls), cname
        for field, _ in cls._fields_:
            assert int(got[f"{cname}.{field}"]) == getattr(cls, field).offset, f"{cname}.{field}"
    assert got["constants"] == f"{native.CACHE_ABI_VERSION}{native.CACHE_PAGE}{native.CACHE_INT8}{native.CACHE_FP8}"


def _good(name):
    """Arguments that pass every check but the last: addresses that no call here reaches."""
    cache = native.PiperCache(4096, 4096, 4096, 4096, 4096, 4096, 8, 2, 64, native.CACHE_INT8)
    rows = native.PiperCacheRows(4096, 4096, None, 4, 4, 3, 5)
    tensor = native.PiperTensor(4096, 640, 320, 64)
    version, dtype = native.CACHE_ABI_VERSION, native.FLOAT16
    if name == "write":
        return native.PiperCacheWriteArgs(version, dtype, cache, rows, tensor, tensor)
    if name == "read":
        return native.PiperCacheReadArgs(version, dtype, cache, rows, 4096, 4096)
    if name == "attention":
        return native.PiperCacheAttentionArgs(version, dtype, 0.125, 0, 4, cache, rows, tensor, None, 0, 0, None, 0, 4096, None, 0)
    return native.PiperCacheSelectArgs(version, dtype, 4, cache, rows, tensor, 2, 4096, None, 0)


@pytest.mark.parametrize("name", ["write", "read", "attention", "select"])
@pytest.mark.parametrize("field, value, message", [
    ("abi_version", 99, "ABI version"),
    ("dtype", native.FLOAT32, "float16 or bfloat16"),
    ("cache.head_dim", 96, "head_dim must be 64 or 128"),
    ("cache.code", 2, "unknown cache code"),
    ("cache.pages", 0, "sizes must be positive"),
    ("cache.pages", 1 << 31, "too large"),
    ("cache.kv_heads", -1, "sizes must be positive"),
    ("rows.batch", 0, "sizes must be positive"),
    ("rows.tokens", 0, "sizes must be positive"),
    ("rows.tokens", 1 << 27, "too large"),
    ("rows.table_width", 0, "sizes must be positive"),
    ("rows.table_width", 1 << 25, "too large"),
    ("rows.page_table", None, "page_table or starts is NULL"),
    ("rows.starts", None, "page_table or starts is NULL"),
    ("rows.table_stride", -4, "table_stride"),
])
def test_c_calls_validate_before_launching(lib, name, field, value, message) -> None:
    args = _good(name)
    at = args
    *outer, last = field.split(".")
    for part in outer:
        at = getattr(at, part)
    setattr(at, last, value)
    with pytest.raises(RuntimeError, match=message):
        lib.cache_call(name, args, 0)


@pytest.mark.parametrize("name, change, message", [
    ("write", {"key": native.PiperTensor(None, 0, 0, 0)}, "key pointer is NULL"),
    ("write", {"value": native.PiperTensor(4100, 0, 0, 0)}, "16-byte aligned"),
    ("write", {"key": native.PiperTensor(4096, 0, 0, 12)}, "multiples of 8"),
    ("read", {"key": None}, "key pointer is NULL"),
    ("read", {"value": 4104}, "16-byte aligned"),
    ("attention", {"heads": 3}, "multiple of kv_heads"),
    ("attention", {"heads": 0}, "multiple of kv_heads"),
    ("attention", {"scale": float("nan")}, "finite and positive"),
    ("attention", {"output": None}, "output pointer is NULL"),
    ("attention", {"query": native.PiperTensor(None, 0, 0, 0)}, "query pointer is NULL"),
    ("attention", {"selected": 4096, "budget": 0}, "budget must be positive"),
    ("attention", {"selected": 4096, "budget": 1, "mask": 4096}, "do not go together"),
    ("attention", {"mask": 4096, "mask_stride_row": -1}, "mask strides"),
    ("select", {"heads": 5}, "multiple of kv_heads"),
    ("select", {"budget": 0}, "budget must be positive"),
    ("select", {"output": None}, "output pointer is NULL"),
])
def test_c_calls_check_their_own_arguments(lib, name, change, message) -> None:
    args = _good(name)
    for field, value in change.items():
        setattr(args, field, value)
    with pytest.raises(RuntimeError, match=message):
        lib.cache_call(name, args, 0)


def test_c_calls_check_the_cache_pointers(lib) -> None:
    for name, fields in (("write", ("key", "key_scale", "value", "value_scale", "bounds", "bound_scale")),
                         ("read", ("key", "key_scale", "value", "value_scale")), ("attention", ("key", "key_scale", "value", "value_scale")),
                         ("select", ("bounds", "bound_scale"))):
        for field in fields:
            bad, aligned = (4098, "4-byte aligned") if field == "bound_scale" else (4100, "16-byte aligned")
            for value, message in ((None, "cache pointer is NULL"), (bad, aligned)):
                args = _good(name)
                setattr(args.cache, field, value)
                with pytest.raises(RuntimeError, match=message):
                    lib.cache_call(name, args, 0)


@pytest.mark.parametrize("name", ["write", "read"])
def test_c_calls_refuse_more_workgroups_than_a_launch_has(lib, name) -> None:
    args = _good(name)
    args.cache.kv_heads, args.rows.batch, args.rows.tokens = 1, 1 << 22, 2  # two pages each
    with pytest.raises(RuntimeError, match="too large for this build"):
        lib.cache_call(name, args, 0)


# ---- index arithmetic --------------------------------------------------------------------------------------------------


def test_every_index_stays_inside(tmp_path) -> None:
    """csrc/cache.h on the CPU over tables with bad entries, negative and far starts and counts beyond the rows: pages
    are inside the cache, the pages touched cover every row once, slots are inside the page, ends inside the table."""
    (tmp_path / "index.cpp").write_text(r"""
#include <cstdio>
#include <set>
#include "cache.h"
using namespace piper;
#define CHECK(x) do { if (!(x)) { printf("line %d: %s (start %ld count %ld tokens %d)\n", __LINE__, #x, (long)start, (long)count, tokens); return 1; } } while (0)
int main() {
  const int32_t table[2][3] = {{2, -1, 4}, {5, 2147483647, -2147483647 - 1}};
  const int64_t all[] = {-2147483647 - 1, -200, -65, -64, -63, -1, 0, 1, 5, 63, 64, 65, 127, 128, 190, 191, 192, 200, 2147483647};
  for (const int64_t start : all)
    for (const int64_t count : all)
      for (const int tokens : {1, 2, 63, 64, 65, 66, 130, 300}) {
        const int32_t starts[2] = {(int32_t)start, (int32_t)start}, counts[2] = {(int32_t)count, (int32_t)count};
        const CacheRows rows{&table[0][0], starts, counts, 3, 5, 3, tokens};
        const int n = rows.count(0);
        CHECK(n == (count < 0 ? 0 : count > tokens ? tokens : count));
        CHECK((CacheRows{&table[0][0], starts, nullptr, 3, 5, 3, tokens}.count(1)) == tokens);
        std::set<int64_t> seen;
        for (int64_t c = 0; c < pages_touched(tokens); ++c) {
          const int64_t logical = floor_page(start) + c;
          const PageRows in = rows_in_page(rows, 0, logical);
          CHECK(in.n >= 0 && in.slot >= 0 && in.slot + in.n <= kPage && in.first >= 0 && in.first + in.n <= n);
          for (int r = 0; r < in.n; ++r) {
            CHECK(start + in.first + r == logical * kPage + in.slot + r);
            CHECK(seen.insert(in.first + r).second);
          }
          for (int b = 0; b < 2; ++b) {
            const int64_t page = rows.page(b, logical);
            CHECK(page == -1 || (page >= 0 && page < rows.pages && logical >= 0 && logical < 3));
          }
        }
        for (int64_t r = 0; r < n; ++r) CHECK(seen.count(r) == (start + r >= 0 ? 1u : 0u));
        for (int64_t r = 0; r < tokens; ++r) {
          const int64_t end = rows.end(0, r), want = start + r + 1;
          CHECK(end == (want < 0 ? 0 : want > 192 ? 192 : want));
        }
      }
  const long start = 0, count = 0;
  const int tokens = 0;
  for (const int d : {64, 128}) {
    std::set<int> offsets;
    for (int slot = 0; slot < 64; ++slot)
      for (int f = 0; f < d; ++f) CHECK(offsets.insert(value_offset(slot, f, d)).second);
    CHECK(*offsets.begin() == 0 && *offsets.rbegin() == 64 * d - 1);
  }
  printf("ok\n");
}
""")
    exe = tmp_path / "index"
    csrc = REPO / "piper-kernels_amd" / "csrc"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-fsanitize=undefined", f"-I{csrc}", str(tmp_path / "index.cpp"), "-o", str(exe)], check=True)
    result = subprocess.run([str(exe)], capture_output=True, text=True)
    assert result.stdout == "ok\n" and result.stderr == "", result.stdout + result.stderr


# ---- the model ----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_the_model_holds_values_to_half_a_step(dtype) -> None:
    """code * scale is within half a code step of the value: a / 254 in INT8; in FP8 2^-4 of the value, or half the
    smallest step 2^-9 of the scale.  Three FP32 roundings come on top, each at most 2^-24 of a value of magnitude up to a:
    x * (L / a), rounded twice, is off by at most 2 * 2^-24 L in codes, 2 * 2^-24 a in values, and the scale's own rounding
    moves code * scale by at most 2^-24 a."""
    x = tokens_of(1, 3, 200, 128, torch.bfloat16, 1).float()
    codes, scale = quantise(x, dtype)
    a = x.abs().amax(-1, keepdim=True)
    off = (codes.float() * scale[..., None] - x).abs()
    half = a / 254 if dtype is torch.int8 else torch.maximum(x.abs() * 2.0**-4, a / 448 * 2.0**-10)
    assert bool((off <= half + 3 * 2.0**-24 * a).all())


def test_the_model_agrees_with_itself() -> None:
    """Tokens written one by one, in a chunk, and over rejected ones leave the same cache; the selection bounds the scores."""
    table = table_of([3, 2], 7, 2)
    key, value = tokens_of(2, 2, 130, 64, torch.float16, 3), tokens_of(2, 2, 130, 64, torch.float16, 4)
    counts = torch.tensor([130, 70], dtype=torch.int32)
    whole, steps = Model(7, 2, 64, torch.int8), Model(7, 2, 64, torch.int8)
    whole.write(key, value, table, torch.zeros(2, dtype=torch.int32), counts)
    for i in range(0, 130, 13):
        now = (counts - i).clamp(0, 13)
        rejected = tokens_of(2, 2, 13, 64, torch.float16, 100 + i)
        if i % 2 == 0 and i + 13 <= 70:
            steps.write(rejected, rejected, table, torch.full((2,), i, dtype=torch.int32), now)
        steps.write(key[:, :, i : i + 13], value[:, :, i : i + 13], table, torch.full((2,), i, dtype=torch.int32), now)
    for a, b in zip(whole.arrays(), steps.arrays()):
        assert torch.equal(a.view(torch.uint8) if a.dtype is not torch.float32 else a, b.view(torch.uint8) if b.dtype is not torch.float32 else b)
    q = tokens_of(2, 4, 1, 64, torch.float16, 5)
    out, _ = whole.attention(q, table, counts - 1)
    picked = whole.select(q, table, counts - 1, None, 9)
    again, _ = whole.attention(q, table, counts - 1, selected=picked)
    assert torch.allclose(out, again, rtol=1e-12, atol=0)  # every page is selected
    assert picked[0, 0, 0].tolist() == [0, 1, 2] + [-1] * 6 and picked[1, 0, 0].tolist() == [0, 1] + [-1] * 7
