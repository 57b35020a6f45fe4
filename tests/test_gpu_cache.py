"""The quantised cache's operators on MI355X against their definition (tests/_cache.py): every code, scale, bound and
selected page equal, attention within the bound of its roundings; slots and rows that are no call's stay as they were,
whatever they hold."""

from __future__ import annotations

import math

import pytest
import torch

from _cache import PAGE, Model, table_of, tokens_of, tree_mask
from _parity import log
from piper_kernels import QuantizedCache, cache_attention, cache_read, cache_select, cache_write, piper_attention
from piper_kernels._hip import library as native

pytestmark = pytest.mark.gpu

INT8, FP8 = torch.int8, torch.float8_e4m3fn
FP16, BF16 = torch.float16, torch.bfloat16


def ints(*values: int) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32)


def on(device, *tensors):
    return tuple(None if t is None else t.to(device) for t in tensors)


def cache_of(model: Model, device) -> QuantizedCache:
    return QuantizedCache(*(a.to(device) for a in model.arrays()))


def same(got: torch.Tensor, want: torch.Tensor, what: str) -> None:
    """Equal bit for bit, any NaN equal to any other."""
    got = got.cpu()
    assert got.shape == want.shape and got.dtype is want.dtype, what
    if want.dtype is FP8:
        got, want = got.view(torch.int8), want.view(torch.int8)
    if want.is_floating_point():
        got, want = torch.nan_to_num(got.float(), nan=1.5e33), torch.nan_to_num(want.float(), nan=1.5e33)
    if not torch.equal(got, want):
        at = (got != want).nonzero()
        first = tuple(at[0].tolist())
        pytest.fail(f"{what}: {len(at)} of {got.numel()} differ, first at {first}: {got[first]} for {want[first]}")


def same_cache(cache: QuantizedCache, model: Model) -> None:
    for name, got, want in zip(cache._fields, cache, model.arrays()):
        same(got, want, name)


def near(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor) -> None:
    off = (got.cpu().double() - want).abs()
    assert bool((off <= bound).all()), f"off by {float((off / bound.clamp(min=1e-300)).max()):.3g} of the bound"


WRITES = [
    # (starts, counts or None, rows, table widths)
    ((0,), None, 1, [1]),  # the first token
    ((63,), None, 1, [1]),  # the one that fills a page
    ((64, 5, 190), None, 1, [2, 1, 3]),  # one token each
    ((0, 0), None, 64, [1, 1]),  # whole pages
    ((7, 60, 128), (130, 0, 9), 130, [3, 1, 3]),  # ragged chunks, one empty
    ((3, 121), (200, 77), 200, [4, 4]),
    ((-70, 100), (150, -3), 150, [2, 2]),  # positions before the first, a negative count
    ((100, 30), (90, 400), 90, [2, 2]),  # past the table, a count beyond the rows
]


@pytest.mark.parametrize("codes", [INT8, FP8], ids=["int8", "fp8"])
@pytest.mark.parametrize("d, heads, dtype, layout", [(64, 3, FP16, "bhtd"), (128, 1, BF16, "bthd"), (128, 5, FP16, "odd"), (64, 2, BF16, "bthd")])
@pytest.mark.parametrize("starts, counts, rows, widths", WRITES)
def test_write_and_read(starts, counts, rows, widths, d, heads, dtype, layout, codes, gfx950_device) -> None:
    log(f"[case] cache write {starts} {counts} {rows} D{d} H{heads} {dtype} {layout} {codes}")
    table = table_of(widths, sum(widths) + 2, 1)
    if len(widths) > 1:
        table[-1, -1] = 99  # outside the cache
    model = Model(sum(widths) + 2, heads, d, codes, fill=2)
    cache = cache_of(model, gfx950_device)
    b = len(starts)
    key, value = (tokens_of(b, heads, rows, d, dtype, seed, layout) for seed in (3, 4))
    key[0, 0, 0] = 0  # a row of zeros, and one that only subnormals stand in
    value[0, -1, 0] = 0
    value[0, -1, 0, 3] = torch.finfo(dtype).smallest_normal / 8
    where = (table, ints(*starts), None if counts is None else ints(*counts))
    model.write(key, value, *where)
    dev = on(gfx950_device, *where)
    cache_write(cache, key.to(gfx950_device), value.to(gfx950_device), *dev)
    same_cache(cache, model)
    got = cache_read(cache, *dev, size=rows, dtype=dtype)
    for x, y, name in zip(got, model.read(*where, rows, dtype), ("key", "value")):
        same(x, y, name)
    # another range, type and size
    shift = ints(*(max(0, s - 3) for s in starts))
    size = rows + 5
    clean = Model(sum(widths) + 2, heads, d, codes)
    clean.write(key, value, *where)
    got = cache_read(cache_of(clean, gfx950_device), dev[0], shift.to(gfx950_device), size=size, dtype=BF16)
    for x, y, name in zip(got, clean.read(table, shift, None, size, BF16), ("key", "value")):
        same(x, y, name)


@pytest.mark.parametrize("codes", [INT8, FP8], ids=["int8", "fp8"])
def test_write_of_what_is_not_finite(codes, gfx950_device) -> None:
    """Infinities and NaN: a NaN scale and zero codes for that row alone; a page's bounds leave it out."""
    log(f"[case] cache write, not finite, {codes}")
    key, value = tokens_of(1, 2, 130, 64, BF16, 5), tokens_of(1, 2, 130, 64, BF16, 6)
    key[0, 0, 3, 7], key[0, 1, 64:128, 5], value[0, 1, 9, 0], value[0, 0, 129, 63] = math.inf, math.nan, -math.inf, math.nan
    value[0, 0, 20] = 2.0**-119  # below what a row is held from
    value[0, 0, 21, :] = 0
    value[0, 0, 21, 4] = 2.0**-118
    table = table_of([3], 4, 7)
    model = Model(4, 2, 64, codes)
    cache = cache_of(model, gfx950_device)
    model.write(key, value, table, ints(0))
    cache_write(cache, *on(gfx950_device, key, value, table, ints(0)))
    same_cache(cache, model)
    assert cache.bound_scale[table[0, 1], 1] == 0 and cache.key_scale.isnan().sum() == 65


ATTENTION = [
    # (starts, counts or None, rows, query heads, kv heads, D, dtype, codes, layout)
    ((0,), None, 1, 1, 1, 64, FP16, INT8, "bhtd"),  # one key
    ((63, 64), None, 1, 4, 2, 128, BF16, FP8, "bhtd"),  # the edges of a page
    ((1000, 3, 517), None, 1, 8, 1, 128, FP16, INT8, "bthd"),
    ((200,), None, 1, 14, 2, 64, BF16, INT8, "odd"),  # a group of seven
    ((130, 0, 700), (5, 0, 7), 7, 6, 2, 64, FP16, FP8, "bhtd"),  # ragged, one without a row
    ((0, 129), None, 70, 2, 2, 128, BF16, INT8, "bthd"),  # a chunk from the start
    ((37, 300), (129, 90), 129, 4, 1, 64, FP16, INT8, "bhtd"),
    ((500,), None, 33, 32, 2, 128, FP16, FP8, "bhtd"),  # sixteen query heads a K/V head
    ((-3, 250), (9, 12), 12, 2, 1, 64, FP16, INT8, "bhtd"),  # rows before the first position see nothing
    ((120,), (200,), 20, 2, 2, 128, BF16, FP8, "bhtd"),  # past the table
]


# more pages than one workgroup takes: parts of a sequence's pages, or shares of all sequences', joined afterwards
LONG = [
    ((2500,), None, 1, 8, 2, 128, BF16, INT8, "bhtd"),
    ((2100,), (3,), 5, 8, 2, 64, FP16, FP8, "bthd"),  # 17 to 32 rows a K/V head, two of five tokens padding
    ((1800,), None, 40, 8, 2, 128, FP16, INT8, "bthd"),  # more than 32
    ((3000, 5, 0, 1700, -20), (1, 1, 0, 1, 1), 1, 6, 2, 64, BF16, INT8, "bhtd"),  # no row, and rows that see nothing
    ((1500, 40, 900), (40, 40, 13), 40, 8, 2, 128, BF16, FP8, "bhtd"),
    (tuple((37 * b * b) % 1300 for b in range(70)), None, 1, 4, 1, 64, FP16, FP8, "bhtd"),  # more sequences than lanes
    (tuple((211 * b) % 1100 for b in range(67)), tuple(b % 4 for b in range(67)), 3, 4, 1, 64, BF16, INT8, "bhtd"),
    ((1100, 1300), None, 130, 2, 2, 64, FP16, INT8, "odd"),
]


def _filled(case, seed: int = 11):
    """A cache that holds a case's tokens among bytes that mean nothing (NaN scales, FP8 NaN codes)."""
    starts, counts, rows, _, heads, d, dtype, codes, _ = case
    b = len(starts)
    real = [rows if counts is None else max(0, min(rows, c)) for c in (counts or [rows] * b)]
    ends = [max(1, s + n) for s, n in zip(starts, real)]
    widths = [-(-e // PAGE) for e in ends]
    if starts == (120,):
        widths = [2]  # the last rows stand past the table
    model = Model(sum(widths) + 1, heads, d, codes, fill=seed)
    table = table_of(widths, sum(widths) + 1, seed)
    longest = max(ends)
    key, value = (tokens_of(b, heads, longest, d, dtype, seed + k) for k in (1, 2))
    model.write(key, value, table, ints(*[0] * b), ints(*ends))
    return model, table, ints(*starts), None if counts is None else ints(*counts)


def _name(case) -> str:
    return str(case) if len(case[0]) < 10 else f"{len(case[0])} sequences {case[2:]}"


@pytest.mark.parametrize("case", ATTENTION + LONG, ids=_name)
def test_attention(case, gfx950_device) -> None:
    log(f"[case] cache attention {case}")
    model, *where = _filled(case)
    starts, counts, rows, hq, _, d, dtype, _, layout = case
    q = tokens_of(len(starts), hq, rows, d, dtype, 20, layout)
    cache, dev = cache_of(model, gfx950_device), on(gfx950_device, *where)
    for scale in (None, 0.31):
        got = cache_attention(q.to(gfx950_device), cache, *dev, scale=scale)
        assert got.is_contiguous() and got.dtype is dtype
        near(got, *model.attention(q, *where, scale=scale))


@pytest.mark.parametrize("case", [c for c in ATTENTION + LONG if c[2] > 1] + [((63,), None, 1, 2, 1, 64, FP16, INT8, "bhtd")], ids=_name)
def test_attention_to_a_tree(case, gfx950_device) -> None:
    log(f"[case] cache attention, tree {case}")
    model, *where = _filled(case, 31)
    starts, _, rows, hq, _, d, dtype, _, layout = case
    b = len(starts)
    q = tokens_of(b, hq, rows, d, dtype, 21, layout)
    cache, dev = cache_of(model, gfx950_device), on(gfx950_device, *where)
    every = tree_mask(b, rows, 22)
    every[0, rows // 2] = False  # a row that sees the cached tokens alone, or nothing
    shared = torch.rand((1, rows, rows), generator=torch.Generator().manual_seed(23)) < 0.4  # no order at all
    view = torch.zeros((b, rows, 2 * rows), dtype=torch.bool)[:, :, ::2]
    view.copy_(every)
    for mask in (every, shared, view, shared.expand(b, rows, rows)):
        got = cache_attention(q.to(gfx950_device), cache, *dev, mask=mask.to(gfx950_device) if mask is not view else _strided(mask, gfx950_device))
        near(got, *model.attention(q, *where, mask=mask))


def _strided(mask, device):
    wide = torch.zeros((*mask.shape[:2], 2 * mask.shape[2]), dtype=torch.bool, device=device)
    wide[:, :, ::2] = mask.to(device)
    return wide[:, :, ::2]


@pytest.mark.parametrize("case", ATTENTION + LONG[:5], ids=_name)
def test_attention_to_selected_pages(case, gfx950_device) -> None:
    """Lists in any order, with pages named twice, pages after the row's own, beyond the table and negative ones."""
    log(f"[case] cache attention, selected {case}")
    model, *where = _filled(case, 41)
    starts, _, rows, hq, heads, d, dtype, _, layout = case
    b = len(starts)
    q = tokens_of(b, hq, rows, d, dtype, 21, layout)
    cache, dev = cache_of(model, gfx950_device), on(gfx950_device, *where)
    for budget in (1, 2, 5, 19, 70):
        g = torch.Generator().manual_seed(budget)
        selected = torch.randint(-1, where[0].shape[1] + 2, (b, heads, rows, budget), generator=g, dtype=torch.int32)
        selected[0, 0, 0] = -1  # nothing at all
        got = cache_attention(q.to(gfx950_device), cache, *dev, selected=selected.to(gfx950_device))
        near(got, *model.attention(q, *where, selected=selected))


@pytest.mark.parametrize("rows", [1, 2, 6, 7, 8, 9, 15, 37])
@pytest.mark.parametrize("heads", [2, 40])
def test_masks_at_every_place_of_a_page(heads, rows, gfx950_device) -> None:
    """Drafted tokens from any slot on, across a page's end, fewer and more than a load of the mask has; any byte but 0
    is true."""
    log(f"[case] cache attention, masks of {rows} rows, {heads} heads")
    starts = (0, 1, 5, 8, 29, 56, 60, 63, 64, 123)
    model, *where = _filled((starts, None, rows, heads, 1, 64, FP16, INT8, "bhtd"), 24)
    q = tokens_of(len(starts), heads, rows, 64, FP16, 25)
    mask = torch.rand((len(starts), rows, rows), generator=torch.Generator().manual_seed(26)) < 0.5
    some = torch.tensor([1, 2, 128, 255], dtype=torch.uint8).repeat(rows * rows)[: rows * rows].view(rows, rows)
    held = (mask.to(torch.uint8) * some).to(gfx950_device).view(torch.bool)
    got = cache_attention(q.to(gfx950_device), cache_of(model, gfx950_device), *on(gfx950_device, *where), mask=held)
    near(got, *model.attention(q, *where, mask=mask))


@pytest.mark.parametrize("batch, rows", [(1, 1), (2, 3), (40, 20)])
def test_lists_shorter_than_their_budget(batch, rows, gfx950_device) -> None:
    """What follows a list's last page is not walked through: lists of every length, in parts and in one."""
    log(f"[case] cache attention, short lists, {batch} x {rows}")
    starts = tuple(600 + 5 * b for b in range(batch))
    model, *where = _filled((starts, None, rows, 6, 2, 64, BF16, INT8, "bhtd"), 43)
    q = tokens_of(batch, 6, rows, 64, BF16, 44)
    cache, dev = cache_of(model, gfx950_device), on(gfx950_device, *where)
    for budget in (3, 64, 65, 130):
        g = torch.Generator().manual_seed(budget)
        selected = torch.randint(0, where[0].shape[1], (batch, 2, rows, budget), generator=g, dtype=torch.int32)
        length = torch.randint(0, budget + 1, (batch, 2, rows, 1), generator=g)
        length[0, 0, 0], length[-1, 1, -1] = 0, budget
        selected = torch.where(torch.arange(budget) < length, selected, -1)
        got = cache_attention(q.to(gfx950_device), cache, *dev, selected=selected.to(gfx950_device))
        near(got, *model.attention(q, *where, selected=selected))


@pytest.mark.parametrize("codes", [INT8, FP8], ids=["int8", "fp8"])
def test_attention_beside_bad_pages_and_what_is_not_finite(codes, gfx950_device) -> None:
    """Table entries outside the cache are not seen; a NaN token makes NaN of the rows that see it and no others."""
    log(f"[case] cache attention, bad pages, {codes}")
    case = ((300,), None, 40, 4, 2, 64, FP16, codes, "bhtd")
    model, table, starts, _ = _filled(case, 51)
    table[0, 1], table[0, 3] = 12345, -7
    q = tokens_of(1, 4, 40, 64, FP16, 52)
    dev = on(gfx950_device, table, starts)
    near(cache_attention(q.to(gfx950_device), cache_of(model, gfx950_device), *dev), *model.attention(q, table, starts))
    every = torch.full_like(table, -1)
    got = cache_attention(q.to(gfx950_device), cache_of(model, gfx950_device), every.to(gfx950_device), dev[1])
    assert bool((got == 0).all())
    # drafted token 17 is not finite: its value in head 0, its key in head 1
    key, value = tokens_of(1, 2, 1, 64, FP16, 53), tokens_of(1, 2, 1, 64, FP16, 54)
    value[0, 0, 0, 3], key[0, 1, 0, 5] = math.nan, math.inf
    model.write(key, value, table, ints(317))
    cache = cache_of(model, gfx950_device)
    mask = tree_mask(1, 40, 55)
    for m in (None, mask):
        got = cache_attention(q.to(gfx950_device), cache, *dev, mask=None if m is None else m.to(gfx950_device)).cpu()
        sees = mask[0, :, 17] if m is not None else torch.arange(40) >= 17
        assert bool(got[0, :, sees].isnan().all()) and bool(got[0, :, ~sees].isfinite().all())
        want, bound = model.attention(q, table, starts, mask=m)
        near(got[:, :, ~sees], want[:, :, ~sees], bound[:, :, ~sees])


@pytest.mark.parametrize("case", ATTENTION, ids=str)
@pytest.mark.parametrize("budget", [1, 2, 4, 40])
def test_select(case, budget, gfx950_device) -> None:
    log(f"[case] cache select {case} {budget}")
    model, *where = _filled(case, 61)
    starts, _, rows, hq, _, d, dtype, _, layout = case
    q = tokens_of(len(starts), hq, rows, d, dtype, 62, layout)
    q[0, 0, 0] = 0
    got = cache_select(q.to(gfx950_device), cache_of(model, gfx950_device), *on(gfx950_device, *where), budget=budget)
    same(got, model.select(q, *where, budget), "selected")


@pytest.mark.parametrize("width, budget, heads", [(700, 33, 2), (1500, 257, 1), (300, 300, 4), (258, 257, 8),
                                                   (1100, 64, 20), (2300, 5, 7), (16384, 500, 1), (17000, 65, 2), (17000, 16999, 1)])
def test_select_among_many(width, budget, heads, gfx950_device) -> None:
    """Many pages, ties among them (pages that the table names again, whose scores are equal), entries outside."""
    log(f"[case] cache select among {width}, {budget}")
    pages = 90
    model = Model(pages, 1, 128, INT8)
    g = torch.Generator().manual_seed(width)
    model.bounds.copy_(torch.randint(-127, 128, model.bounds.shape, generator=g))
    model.bound_scale.copy_(torch.rand(model.bound_scale.shape, generator=g))
    table = torch.randint(0, pages, (2, width), generator=g, dtype=torch.int32)
    table[0, 5], table[1, 7] = -1, pages
    q = tokens_of(2, heads, 3, 128, BF16, 63)
    where = (table, ints(width * PAGE - 3, (width - 9) * PAGE - 2), None)
    got = cache_select(q.to(gfx950_device), cache_of(model, gfx950_device), *on(gfx950_device, *where), budget=budget)
    same(got, model.select(q, *where, budget), "selected")


@pytest.mark.parametrize("width", [1, 16, 63, 64, 65])
@pytest.mark.parametrize("heads", [1, 3, 8, 20])
def test_select_of_many_rows_among_few(width, heads, gfx950_device) -> None:
    """Short tables, a chunk's rows: also rows that the table does not reach, and a count that ends among a wave's."""
    log(f"[case] cache select of many rows among {width}, {heads}")
    model = Model(70, 1, 64, INT8)
    g = torch.Generator().manual_seed(width)
    model.bounds.copy_(torch.randint(-127, 128, model.bounds.shape, generator=g))
    model.bound_scale.copy_(torch.rand(model.bound_scale.shape, generator=g))
    table = torch.randint(0, 70, (3, width), generator=g, dtype=torch.int32)
    where = (table, ints(width * PAGE - 45, -3, max(0, width * PAGE - 90)), ints(81, 50, 41))
    q = tokens_of(3, heads, 81, 64, BF16, 64)
    dev = on(gfx950_device, *where)
    for budget in (1, 2, width // 2 + 1, width + 3):
        got = cache_select(q.to(gfx950_device), cache_of(model, gfx950_device), *dev, budget=budget)
        same(got, model.select(q, *where, budget), "selected")


@pytest.mark.parametrize("width, heads, rows", [(66, 16, 2101), (66, 3, 4500), (65, 32, 1100), (64, 16, 2101), (1024, 16, 1050)])
def test_select_of_a_long_chunk(width, heads, rows, gfx950_device) -> None:
    """More rows than workgroups: several tiles' rows in each, and the last of them ends early."""
    log(f"[case] cache select of {rows} rows among {width}, {heads} heads")
    model = Model(70, 1, 64, INT8)
    g = torch.Generator().manual_seed(width + rows)
    model.bounds.copy_(torch.randint(-127, 128, model.bounds.shape, generator=g))
    model.bound_scale.copy_(torch.rand(model.bound_scale.shape, generator=g))
    table = torch.randint(0, 70, (1, width), generator=g, dtype=torch.int32)
    where = (table, ints(width * PAGE - rows + 7), ints(rows - 3))
    q = tokens_of(1, heads, rows, 64, BF16, 65)
    got = cache_select(q.to(gfx950_device), cache_of(model, gfx950_device), *on(gfx950_device, *where), budget=9)
    same(got, model.select(q, *where, 9), "selected")


@pytest.mark.parametrize("width, tokens", [(40, 3), (600, 1), (17000, 1)])
def test_select_with_what_is_not_finite(width, tokens, gfx950_device) -> None:
    """Heads that are not finite do not count; where none is left, and where a page's scale is any NaN, scores are -inf."""
    log(f"[case] cache select, not finite, {width}")
    model = Model(30, 2, 64, INT8)
    g = torch.Generator().manual_seed(width)
    model.bounds.copy_(torch.randint(-127, 128, model.bounds.shape, generator=g))
    model.bound_scale.copy_(torch.rand(model.bound_scale.shape, generator=g))
    for page, bits in ((3, -1), (8, 0x7FC00000), (11, 0x7F800001), (20, -0x400000)):
        model.bound_scale[page, 0] = torch.tensor(bits, dtype=torch.int32).view(torch.float32)
    table = torch.randint(0, 30, (1, width), generator=g, dtype=torch.int32)
    where = (table, ints(width * PAGE - tokens), None)
    q = tokens_of(1, 6, tokens, 64, FP16, 66)
    q[0, 1, 0, 5] = math.inf  # one head of the first K/V head
    q[0, 3:6, 0, 2] = math.nan  # every head of the second
    dev = on(gfx950_device, *where)
    for budget in (2, width // 2, width - 1):
        got = cache_select(q.to(gfx950_device), cache_of(model, gfx950_device), *dev, budget=budget)
        same(got, model.select(q, *where, budget), "selected")


@pytest.mark.parametrize("codes", [INT8, FP8], ids=["int8", "fp8"])
@pytest.mark.parametrize("d", [64, 128])
def test_read_rounds_the_product(d, codes, gfx950_device) -> None:
    """FP16 reads: code * scale rounded to FP32 and then to FP16, where one rounding of the two gives another value.
    Scales are made such that for code 3 the exact product is just beside a tie of FP16 and its FP32 value is the tie."""
    log(f"[case] cache read, ties, D{d} {codes}")
    tie = torch.arange(1024, 2048, dtype=torch.float64) + 0.5  # between two halves, in [1024, 2048)
    scale = (tie / 3).float()
    exact, single = scale.double() * 3, scale * 3
    apart = (exact != tie) & (single.double() == tie)
    scale = scale[apart][: 4 * PAGE]
    assert len(scale) == 4 * PAGE
    once = torch.from_numpy((scale.double() * 3).numpy().astype("float16"))
    assert int((once != (scale * 3).half()).sum()) > 50
    cache = QuantizedCache.allocate(4, 1, d, dtype=codes, device=gfx950_device)
    three = torch.tensor(3.0).to(codes).view(torch.int8).item()
    cache.key.view(torch.int8).fill_(three)
    cache.value.view(torch.int8).fill_(three)
    cache.key_scale.copy_(scale.view(4, 1, PAGE))
    cache.value_scale.copy_(scale.view(4, 1, PAGE))
    table = torch.arange(4, dtype=torch.int32, device=gfx950_device)[None]
    want = (scale * 3).half()[None, None, :, None].expand(1, 1, 4 * PAGE, d)
    for x, name in zip(cache_read(cache, table, torch.zeros(1, dtype=torch.int32, device=gfx950_device), size=4 * PAGE, dtype=FP16), ("key", "value")):
        same(x, want, name)


def test_layers_of_one_allocation(gfx950_device) -> None:
    """The layers of a model as slices of one cache, odd numbers of pages and heads among them."""
    log("[case] cache layers")
    layers, pages, d = 3, 3, 64
    whole = QuantizedCache.allocate(layers * pages, 1, d, device=gfx950_device)
    table, starts = torch.tensor([[2, 0]], dtype=torch.int32), ints(0)
    dev = on(gfx950_device, table, starts)
    for layer in range(layers):
        cache = QuantizedCache(*(a[layer * pages : (layer + 1) * pages] for a in whole))
        model = Model(pages, 1, d, INT8)
        key, value = (tokens_of(1, 1, 100, d, BF16, 70 + 2 * layer + i) for i in (0, 1))
        cache_write(cache, key.to(gfx950_device), value.to(gfx950_device), *dev)
        model.write(key, value, table, starts)
        same_cache(cache, model)
        q = tokens_of(1, 2, 100, d, BF16, 90 + layer)
        same(cache_select(q.to(gfx950_device), cache, *dev, budget=1), model.select(q, table, starts, None, 1), "selected")


def test_sizes_that_no_launch_has(gfx950_device) -> None:
    """The workspace functions read no pointer and launch nothing."""
    lib = native.load_library()
    cache = native.PiperCache(pages=64, kv_heads=1, head_dim=64, code=native.CACHE_INT8)
    args_of = {"attention": native.PiperCacheAttentionArgs, "select": native.PiperCacheSelectArgs}

    def bytes_of(name: str, heads: int, batch: int, tokens: int, width: int, **more) -> int:
        rows = native.PiperCacheRows(table_stride=width, table_width=width, batch=batch, tokens=tokens)
        args = args_of[name](abi_version=native.CACHE_ABI_VERSION, dtype=native.FLOAT16, heads=heads, cache=cache, rows=rows, **more)
        return lib.cache_workspace_bytes(name, args)

    assert bytes_of("attention", 8, 2, 4096, 1024) > 0  # shares of a line of blocks' pages
    assert bytes_of("attention", 8, 2, 4096, 1 << 24) == 0  # whose length 32 bits do not hold: a workgroup a block
    for name, sizes, more in (("attention", (1, 1 << 23, 1, 4), {}), ("attention", (1, 1 << 10, 1 << 13, 4), {"selected": 4096, "budget": 2}),
                              ("select", (16, 1 << 13, 1 << 10, 64), {"budget": 2}), ("select", (1, 1 << 13, 4, 1 << 16), {"budget": 2})):
        with pytest.raises(RuntimeError, match="too large for this build"):
            bytes_of(name, *sizes, **more)


def test_a_cache_beyond_32_bits(gfx950_device) -> None:
    """Pages whose bytes start beyond 2^32: written, read, attended to and selected."""
    log("[case] cache beyond 32 bits")
    pages, heads, d = 70000, 8, 128  # 4.6 GB of keys
    cache = QuantizedCache.allocate(pages, heads, d, device=gfx950_device)
    model = Model(3, heads, d, INT8)
    small, far = torch.tensor([[2, 0, 1]], dtype=torch.int32), torch.tensor([[69999, 66000, 69998]], dtype=torch.int32)
    key, value = tokens_of(1, heads, 150, d, BF16, 71), tokens_of(1, heads, 150, d, BF16, 72)
    model.write(key, value, small, ints(0))
    dev = on(gfx950_device, far, ints(0))
    cache_write(cache, *on(gfx950_device, key, value), *dev)
    for x, y in zip(cache_read(cache, *dev, size=150), model.read(small, ints(0), None, 150, BF16)):
        same(x, y, "read")
    q = tokens_of(1, 16, 1, d, BF16, 73)
    at = ints(149).to(gfx950_device)
    near(cache_attention(q.to(gfx950_device), cache, dev[0], at), *model.attention(q, small, ints(149)))
    same(cache_select(q.to(gfx950_device), cache, dev[0], at, budget=2), model.select(q, small, ints(149), None, 2), "selected")
    assert int(cache.key.view(torch.int8)[:66000].count_nonzero()) == 0


def _generate(device, codes, steps=3):
    """A prompt, steps of one token, a drafted tree of which a part is accepted, and steps over selected pages."""
    b, hq, h, d, prompt = 2, 8, 2, 64, 150
    table = table_of([5, 5], 11, 81)
    model, cache = Model(11, h, d, codes), QuantizedCache.allocate(11, h, d, dtype=codes, device=device)
    dev_table = table.to(device)
    lengths = torch.tensor([prompt, 100], dtype=torch.int32)
    key, value = tokens_of(b, h, prompt, d, FP16, 82), tokens_of(b, h, prompt, d, FP16, 83)
    zero = ints(0, 0)
    model.write(key, value, table, zero, lengths)
    cache_write(cache, *on(device, key, value), dev_table, *on(device, zero, lengths))
    yield model, cache, table, lengths, None, None, None
    seed = 90
    for step in range(steps):
        for tokens, mask, accepted in ((1, None, 1), (7, tree_mask(b, 7, seed), 2), (40, None, 40)):
            seed += 5
            k, v, q = (tokens_of(b, heads, tokens, d, FP16, seed + j) for j, heads in enumerate((h, h, hq)))
            model.write(k, v, table, lengths)
            where = on(device, lengths)
            cache_write(cache, *on(device, k, v), dev_table, *where)
            out = cache_attention(q.to(device), cache, dev_table, *where, mask=None if mask is None else mask.to(device))
            picked = cache_select(q.to(device), cache, dev_table, *where, budget=2)
            some = cache_attention(q.to(device), cache, dev_table, *where, selected=picked)
            yield model, cache, table, lengths.clone(), (q, mask), (out, some), picked
            lengths += accepted


@pytest.mark.parametrize("codes", [INT8, FP8], ids=["int8", "fp8"])
def test_a_run_of_them_together(codes, gfx950_device) -> None:
    """Generation as a program does it, every step's cache, output and selection against the definition; the prompt read
    back is what piper_attention takes, and its own attention over the same tokens agrees."""
    log(f"[case] cache, a run of them together, {codes}")
    for model, cache, table, lengths, asked, outs, picked in _generate(gfx950_device, codes):
        same_cache(cache, model)
        if asked is None:
            key, value = cache_read(cache, table.to(gfx950_device), ints(0, 0).to(gfx950_device), size=100, dtype=FP16)
            q = tokens_of(2, 2, 100, 64, FP16, 84)
            ours = cache_attention(q.to(gfx950_device), cache, *on(gfx950_device, table, ints(0, 0)))
            theirs = piper_attention(q.to(gfx950_device), key, value, is_causal=True)
            # the reference's own envelope between 8-bit attention and exact attention: mean 0.01 of unit values
            assert float((ours.float() - theirs.float()).abs().mean()) < 0.01 * float(value.float().abs().max())
            continue
        q, mask = asked
        near(outs[0], *model.attention(q, table, lengths, mask=mask))
        same(picked, model.select(q, table, lengths, None, 2), "selected")
        near(outs[1], *model.attention(q, table, lengths, selected=picked.cpu()))


def test_streams_and_freed_inputs(gfx950_device) -> None:
    """Calls on a side stream whose inputs are freed at once, against the same calls on the current one."""
    log("[case] cache on a side stream")
    case = ((700, 200), None, 9, 8, 2, 128, BF16, INT8, "odd")
    model, *where = _filled(case, 101)
    dev = on(gfx950_device, *where)
    key, value, q = (tokens_of(2, n, 9, 128, BF16, 102 + i, "odd").to(gfx950_device) for i, n in enumerate((2, 2, 8)))
    cache, other = cache_of(model, gfx950_device), cache_of(model, gfx950_device)

    def calls(c, k, v, query):
        cache_write(c, k, v, *dev)
        pages = cache_select(query, c, *dev, budget=4)
        return (cache_attention(query, c, *dev), cache_attention(query, c, *dev, selected=pages), pages, *cache_read(c, *dev, size=9))

    want = calls(cache, key, value, q)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        inputs = [x.clone() for x in (key, value, q)]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = calls(other, *inputs)
        del inputs
        junk = [torch.full_like(key, 7.0) for _ in range(4)]  # takes the freed memory, were it free already
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            same(x, y.cpu(), "side stream")
        del junk, got


def test_graphs(gfx950_device) -> None:
    """A step captured once and replayed with other tables, positions and tokens; two graphs of one cache in turn, eager
    calls between them: every replay equals the eager calls."""
    log("[case] cache steps in graphs")
    b, hq, h, d = 3, 8, 2, 128
    table = table_of([40, 40, 40], 121, 111)
    model = Model(121, h, d, INT8)
    model.write(*(tokens_of(b, h, 2560, d, BF16, s) for s in (112, 113)), table, ints(0, 0, 0))
    cache, eager = cache_of(model, gfx950_device), cache_of(model, gfx950_device)
    table_d, starts = table.to(gfx950_device), ints(5, 0, 9).to(gfx950_device)
    key, value, q = (torch.empty((b, n, 1, d), dtype=BF16, device=gfx950_device).normal_() for n in (h, h, hq))

    def step(c):
        cache_write(c, key, value, table_d, starts)
        pages = cache_select(q, c, table_d, starts, budget=5)
        return cache_attention(q, c, table_d, starts), cache_attention(q, c, table_d, starts, selected=pages), pages, *cache_read(c, table_d, starts, size=1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache)
        step(eager)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(cache)
        graphs.append((graph, out))
    for replay in range(6):
        g = torch.Generator().manual_seed(replay)
        for x, heads in ((key, h), (value, h), (q, hq)):
            x.copy_(torch.randn((b, heads, 1, d), generator=g))
        starts.copy_(torch.randint(0, 2560, (b,), generator=g).int())
        graph, out = graphs[replay % 2]
        graph.replay()
        want = step(eager)
        torch.cuda.synchronize()
        for x, y in zip(out, want):
            same(x, y.cpu(), f"replay {replay}")
        for x, y, name in zip(cache, eager, cache._fields):
            same(x, y.cpu(), name)


def test_compiled(gfx950_device) -> None:
    """The ops in a compiled program, the cache changed in place, against the eager calls."""
    log("[case] cache compiled")
    case = ((300, 70), None, 3, 4, 2, 64, FP16, INT8, "bhtd")
    model, *where = _filled(case, 121)
    table, starts, _ = on(gfx950_device, *where)
    key, value, q = (tokens_of(2, n, 3, 64, FP16, 122 + i).to(gfx950_device) for i, n in enumerate((2, 2, 4)))
    caches = [cache_of(model, gfx950_device) for _ in range(2)]

    def program(arrays, k, v, query):
        c = QuantizedCache(*arrays)
        cache_write(c, k * 2, v, table, starts)
        pages = cache_select(query, c, table, starts, budget=3)
        return cache_attention(query, c, table, starts), cache_attention(query, c, table, starts, selected=pages) + 1, cache_read(c, table, starts, size=3, dtype=FP16)[0]

    with torch.no_grad():
        want = program(tuple(caches[0]), key, value, q)
        got = torch.compile(program, backend="aot_eager", fullgraph=True)(tuple(caches[1]), key, value, q)
    for x, y in zip(got, want):
        same(x, y.cpu(), "compiled")
    for x, y, name in zip(*caches, caches[0]._fields):
        same(x, y.cpu(), name)


def test_calls_leave_their_inputs(gfx950_device) -> None:
    """Nothing but the cache in a write changes, and two calls give the same bits."""
    log("[case] cache inputs and repeats")
    case = ((1900, 17), (6, 3), 6, 16, 4, 128, BF16, FP8, "bhtd")
    model, *where = _filled(case, 131)
    q, mask = tokens_of(2, 16, 6, 128, BF16, 132), tree_mask(2, 6, 133)
    dev = on(gfx950_device, q, mask, *where)
    kept = [x.clone() for x in dev]
    cache = cache_of(model, gfx950_device)
    once = [f() for _ in range(2) for f in (
        lambda: cache_attention(dev[0], cache, *dev[2:], mask=dev[1]), lambda: cache_select(dev[0], cache, *dev[2:], budget=9),
        lambda: cache_read(cache, *dev[2:], size=6)[1])]
    for x, y in zip(once[:3], once[3:]):
        same(x, y.cpu(), "twice")
    same_cache(cache, model)
    for x, y in zip(dev, kept):
        same(x, y.cpu(), "inputs")
