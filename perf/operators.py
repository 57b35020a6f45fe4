"""The quantised KV cache's operators as a generating program calls them: their inputs, plain forms and costs.

The cache is paged, 64 tokens a page, K and V in 8 bits with an FP32 scale per token and head (``QuantizedCache``'s
documented layout, which the plain form reads and writes too).  A case is one pass: tokens written and read back, a
prefix read, attention over the cache (one token, a drafted tree, a chunk of a prompt, or over selected pages), or the
selection of pages.  ``own`` false runs elementary torch operations, true the package's operators.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

PAGE = 64
_TINY = 2.0**-118  # a row whose largest magnitude is below this is held as zeros
_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_CODES = {"int8": (torch.int8, 127.0), "fp8": (torch.float8_e4m3fn, 448.0)}


def _case(name, op, batch, heads, kv_heads, d, tokens, context, dtype, codes, *, ragged=False, layout="bhtd", budget=0):
    """``tokens`` new tokens a sequence (for "read": tokens read) after ``context`` cached ones."""
    case = {"op": op, "batch": batch, "heads": heads, "kv_heads": kv_heads, "d": d, "tokens": tokens, "context": context,
            "dtype": dtype, "codes": codes, "ragged": ragged, "layout": layout, "budget": budget}
    return {"name": name, **case} if name else case


def listed():
    return [
        # the token of each running request, all latency
        _case("write-step", "write", 64, 32, 8, 128, 1, 8191, "bf16", "int8", ragged=True),
        # prompts entering the cache, from projections that keep a token's heads together
        _case("write-prompt", "write", 4, 32, 8, 128, 8192, 0, "bf16", "fp8", layout="bthd"),
        # a short ragged prefix of a small model read back for the next chunk's attention
        _case("read-ragged-d64", "read", 3, 8, 8, 64, 1001, 37, "fp16", "int8", ragged=True),
        # long prefixes read back
        _case("read-long", "read", 4, 32, 8, 128, 32768, 0, "bf16", "fp8"),
        # the smallest attention call: one token of one short sequence
        _case("step-small-d64", "attention", 1, 8, 8, 64, 1, 334, "fp16", "int8"),
        # one token each of a full batch of requests of every length
        _case("step-batch", "attention", 64, 32, 8, 128, 1, 8191, "bf16", "int8", ragged=True),
        # one token of one very long sequence (the length of workload r2)
        _case("step-long", "attention", 1, 32, 8, 128, 1, 131071, "bf16", "fp8"),
        # trees of drafted tokens of a batch, to be verified in one pass
        _case("tree", "tree", 8, 32, 8, 128, 61, 8192, "fp16", "int8", ragged=True, layout="bthd"),
        # a chunk of a long prompt
        _case("chunk", "attention", 1, 32, 8, 128, 2048, 32768, "bf16", "int8"),
        # pages for one token each of long requests
        _case("select-step", "select", 16, 32, 8, 128, 1, 65535, "bf16", "int8", ragged=True, budget=64),
        # pages for every token of a chunk
        _case("select-chunk", "select", 1, 16, 4, 64, 500, 16384, "fp16", "fp8", budget=32),
        # attention of those steps over their selected pages
        _case("selected-step", "selected", 16, 32, 8, 128, 1, 65535, "bf16", "int8", ragged=True, budget=64),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """Every pass, both head sizes, code types, dtypes and layouts; 1 to 64 sequences, contexts up to 131072, 1 to 8192
    tokens, 1 to 16 query heads a K/V head; at most the cost of the largest listed cases."""
    while True:
        op = rng.choice(("write", "read", "attention", "attention", "tree", "select", "selected"))
        batch, kv_heads = _log_uniform(rng, 1, 64), rng.choice((1, 2, 4, 5, 8, 16))
        heads = kv_heads * rng.choice((1, 2, 4, 4, 7, 8, 16))
        context = _log_uniform(rng, 1, 131072)
        form = rng.random()
        tokens = 1 if form < 0.4 else _log_uniform(rng, 2, 100) if form < 0.8 else _log_uniform(rng, 64, 8192)
        if op == "read":
            tokens, context = _log_uniform(rng, 1, 32768), rng.choice((0, 0, rng.randrange(1000)))
        if op == "tree":
            tokens = _log_uniform(rng, 2, 128)
        budget = _log_uniform(rng, 1, 128) if op in ("select", "selected") else 0
        case = _case(None, op, batch, heads, kv_heads, rng.choice((64, 128, 128)), tokens, context, rng.choice(("fp16", "bf16")),
                     rng.choice(("int8", "fp8")), ragged=rng.random() < 0.6, layout=rng.choice(("bhtd", "bhtd", "bthd")), budget=budget)
        cost = work(case)
        rows = batch * heads * tokens
        held = batch * kv_heads * (context + tokens) * case["d"] * 2
        # what the plain form holds in FP32: scores of every key, or the selected pages' keys and values
        plain = rows * (context + tokens) if op in ("attention", "tree") else 0
        if op == "select":
            plain = rows * (context + tokens) // PAGE * 4
        if op == "selected":
            plain = batch * kv_heads * tokens * budget * PAGE * case["d"]
        if cost["flops"] <= 1.2e12 and cost["bytes"] <= 1.1e9 and held <= 2.2e9 and plain <= 2.4e9:
            return case


# ---- inputs ---------------------------------------------------------------------------------------------------------


def _lengths(case, g):
    """(starts, counts) of the sequences: all alike, or ragged with the first the longest."""
    b = case["batch"]

    def some(most, least):
        x = torch.full((b,), most, dtype=torch.int32)
        if case["ragged"]:
            x = (least + torch.rand(b, generator=g) * (most + 1 - least)).int().clamp_(max=most)
            x[0] = most
        return x

    return some(case["context"], case["context"] // 4), some(case["tokens"], min(1, case["tokens"]))


def _tokens(case, heads, g, bias=None, spread=0.0):
    b, t, d = case["batch"], case["tokens"], case["d"]
    x = torch.randn((b, heads, t, d), generator=g, device="cuda")
    if bias is not None:
        x += bias
    if spread:
        x *= torch.exp(spread * torch.randn((b, heads, t, 1), generator=g, device="cuda"))
    x = x.to(_DTYPES[case["dtype"]])
    return x if case["layout"] == "bhtd" else x.transpose(1, 2).contiguous().transpose(1, 2)


def _quantise(x, codes):
    """(codes, scales) of FP32 rows: scale = a / L, code = round(x * (L / a)) with a the row's largest magnitude."""
    kind, largest = _CODES[codes]
    a = x.abs().amax(-1, keepdim=True)
    top = torch.full((), largest, device=x.device)  # a tensor: a number would be divided by as a product
    zero = a < _TINY
    scaled = x * torch.where(zero, torch.zeros_like(a), top / torch.where(zero, top, a))
    if codes == "int8":
        scaled = scaled.round()
    return scaled.clamp(-largest, largest).to(kind), torch.where(zero, torch.zeros_like(a), a / top).squeeze(-1)


def _bounds(key):
    """(bounds, bound_scale) of pages of dequantised keys [..., 64, D]."""
    ends = torch.stack((key.amax(-2), key.amin(-2)), -2)
    codes, scale = _quantise(ends.flatten(-2), "int8")
    return codes.view(ends.shape), scale


def _pages(case, starts, counts, g, bias):
    """A cache that holds the sequences' tokens, its pages in no order, and the table that says where they are."""
    b, h, d, codes = case["batch"], case["kv_heads"], case["d"], case["codes"]
    total = (starts + counts + PAGE - 1) // PAGE
    width = int(total.max())
    n = b * width + 1  # the pages that requests of full length need, and one
    order = torch.randperm(n, generator=g).int()
    table = torch.where(torch.arange(width)[None] < total[:, None], order[:-1].view(b, width), torch.full((), -1, dtype=torch.int32))
    gg = torch.Generator(device="cuda").manual_seed(int(order.sum()) % 65521 + int(g.initial_seed()))

    def rows(offset):
        x = torch.randn((n, h, PAGE, d), generator=gg, device="cuda")
        x += offset
        x *= torch.exp(0.3 * torch.randn((n, h, PAGE, 1), generator=gg, device="cuda"))
        return _quantise(x, codes)

    key, key_scale = rows(bias)
    bounds, bound_scale = _bounds(key.float() * key_scale[..., None])
    value, value_scale = rows(0.5)
    # token 8a + j, feature d at [a, d, j]
    value = value.view(torch.int8).view(n, h, 8, 8, d).transpose(-1, -2).contiguous().view(value.dtype)
    cache = {"key": key, "key_scale": key_scale, "value": value, "value_scale": value_scale, "bounds": bounds, "bound_scale": bound_scale}
    return cache, table.cuda()


def _tree(case, g):
    """mask[b, i, j]: drafted token j is i or an ancestor of i; each node's parent stands before it."""
    b, t = case["batch"], case["tokens"]
    mask = torch.zeros((b, t, t), dtype=torch.bool)
    near = torch.rand((b, t), generator=g)
    every = torch.arange(b)
    for i in range(t):
        if i:
            parent = i - 1 - (near[:, i] ** 2 * min(i, 8)).long().clamp(max=min(i, 8) - 1)
            mask[:, i] = mask[every, parent]
        mask[:, i, i] = True
    return mask.cuda()


def _selected(case, starts, g):
    """Pages a selection would give: the own page and distinct earlier ones, ascending, -1 behind them."""
    b, h, t, k = case["batch"], case["kv_heads"], case["tokens"], case["budget"]
    page = (starts.cuda()[:, None] + torch.arange(t, device="cuda")[None]) // PAGE
    n = int(page.max()) + 1
    gg = torch.Generator(device="cuda").manual_seed(int(g.initial_seed()) + 17)
    score = torch.rand((b, h, t, n), generator=gg, device="cuda")
    at = torch.arange(n, device="cuda")
    score = torch.where(at > page[:, None, :, None], -1.0, torch.where(at == page[:, None, :, None], 2.0, score))
    best, index = score.topk(min(k, n), -1)
    index = torch.where(best < 0, n, index).sort(-1).values
    out = torch.full((b, h, t, k), -1, dtype=torch.int32, device="cuda")
    out[..., : index.shape[-1]] = torch.where(index == n, -1, index)
    return out


def prepare(case, seed):
    g = torch.Generator().manual_seed(seed)
    gg = torch.Generator(device="cuda").manual_seed(seed)
    starts, counts = _lengths(case, g)
    bias = math.sqrt(2.0) * torch.randn((case["kv_heads"], 1, case["d"]), generator=gg, device="cuda")  # what trained keys show
    cache, table = _pages(case, starts, counts, g, bias)
    state = {"op": case["op"], "codes": case["codes"], "cache": cache, "table": table, "starts": starts.cuda(), "counts": counts.cuda(),
             "tokens": case["tokens"], "budget": case["budget"], "dtype": _DTYPES[case["dtype"]]}
    if case["op"] == "write":
        state["key"] = _tokens(case, case["kv_heads"], gg, bias, 0.3)
        state["value"] = _tokens(case, case["kv_heads"], gg, 0.5, 0.3)
    elif case["op"] != "read":
        state["query"] = _tokens(case, case["heads"], gg)
    if case["op"] == "tree":
        state["mask"] = _tree(case, g)
    if case["op"] == "selected":
        state["selected"] = _selected(case, starts, g)
    return state


# ---- one pass ---------------------------------------------------------------------------------------------------------


def run(state):
    op, cache = state["op"], state["cache"]
    where = (state["table"], state["starts"], state["counts"])
    if own:
        try:
            from piper_kernels import QuantizedCache, cache_attention, cache_read, cache_select, cache_write
        except ImportError:  # the first call
            sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "piper-kernels_amd"))
            from piper_kernels import QuantizedCache, cache_attention, cache_read, cache_select, cache_write

        cache = QuantizedCache(**cache)
        if op == "write":
            cache_write(cache, state["key"], state["value"], *where)
        if op in ("write", "read"):
            key, value = cache_read(cache, *where, size=state["tokens"], dtype=state["dtype"])
        elif op == "select":
            return cache_select(state["query"], cache, *where, budget=state["budget"])
        else:
            return cache_attention(state["query"], cache, *where, mask=state.get("mask"), selected=state.get("selected"))
    else:
        if op == "write":
            _plain_write(state)
        if op in ("write", "read"):
            key, value = _plain_read(state)
        elif op == "select":
            return _plain_select(state)
        elif op == "selected":
            return _plain_selected(state)
        else:
            return _plain_attention(state)
    # the 8-bit K and V come as the values they stand for, by the read; a page's bounds have no reader but the selection
    # and come as they are held, which has to be equal to the bit
    return {"key": key, "value": value, "bounds": cache["bounds"] if not own else cache.bounds,
            "bound_scale": cache["bound_scale"] if not own else cache.bound_scale} if op == "write" else {"key": key, "value": value}


def _slots(state):
    """Positions of the rows [B, T], which are real, and their page and slot."""
    i = torch.arange(state["tokens"], device="cuda")[None]
    real = i < state["counts"][:, None]
    position = state["starts"][:, None] + torch.where(real, i, 0)  # a row that is none stands for the first
    page = state["table"].gather(1, (position // PAGE).long())
    return position, real, page, position % PAGE


def _plain_write(state):
    cache, codes = state["cache"], state["codes"]
    _, real, page, slot = _slots(state)
    i = torch.where(real, torch.arange(state["tokens"], device="cuda")[None], 0)
    for name in ("key", "value"):
        x = state[name].transpose(1, 2).float()  # [B, T, H, D]
        c, s = _quantise(x.gather(1, i[..., None, None].expand_as(x)), codes)
        c, at, scale = c.view(torch.int8), cache[name].view(torch.int8), cache[name + "_scale"]
        if name == "value":
            at[page, :, slot // 8, :, slot % 8] = c
        else:
            at[page, :, slot] = c
        scale[page, :, slot] = s
    # bounds of the pages that these tokens fill
    first = state["starts"][:, None] // PAGE
    last = (state["starts"] + state["counts"] - 1)[:, None] // PAGE
    logical = torch.minimum(first + torch.arange(state["tokens"] // PAGE + 2, device="cuda")[None], last)
    page = state["table"].gather(1, logical.long())
    full = ((logical + 1) * PAGE <= (state["starts"] + state["counts"])[:, None])[..., None]
    bounds, scale = _bounds(cache["key"][page].float() * cache["key_scale"][page][..., None])
    cache["bounds"][page] = torch.where(full[..., None, None], bounds, cache["bounds"][page])
    cache["bound_scale"][page] = torch.where(full, scale, cache["bound_scale"][page])


def _plain_read(state):
    cache = state["cache"]
    _, real, page, slot = _slots(state)
    out = []
    for name in ("key", "value"):
        held = cache[name].view(torch.int8)
        c = held[page, :, slot // 8, :, slot % 8] if name == "value" else held[page, :, slot]
        x = c.view(cache[name].dtype).float() * cache[name + "_scale"][page, :, slot][..., None]  # [B, T, H, D]
        out.append(torch.where(real[..., None, None], x, 0.0).to(state["dtype"]).transpose(1, 2).contiguous())
    return out


def _page_values(cache, page, head=slice(None)):
    """Keys and values [..., 64, D] of pages in FP32."""
    key = cache["key"][page, head].float() * cache["key_scale"][page, head][..., None]
    value = cache["value"][page, head].float().transpose(-1, -2).flatten(-3, -2) * cache["value_scale"][page, head][..., None]
    return key, value


def _soft(scores, visible, value):
    s = scores.masked_fill_(~visible, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, value) / torch.where(total == 0, 1.0, total)


def _plain_attention(state):
    q, table, starts, counts = state["query"], state["table"], state["starts"], state["counts"]
    b, hq, t, d = q.shape
    key, value = (x.transpose(1, 2).flatten(2, 3) for x in _page_values(state["cache"], table.clamp(min=0)))  # [B, H, S, D]
    h = key.shape[1]
    scores = torch.matmul((q.float() * d**-0.5).reshape(b, h, hq // h * t, d), key.transpose(-1, -2).contiguous())
    j = torch.arange(key.shape[2], device="cuda")[None, None]
    draft = j - starts[:, None, None]  # [B, 1, S]
    i = torch.arange(t, device="cuda")[None, :, None]
    if "mask" in state:
        seen = state["mask"].gather(2, draft.clamp(0, t - 1).expand(b, t, -1).long())
        visible = (draft < 0) | (seen & (draft < counts[:, None, None]) & (draft < t))
    else:
        visible = draft <= i
    real = i < counts[:, None, None]
    visible = (visible & real)[:, None, None].expand(b, 1, hq // h, t, -1).reshape(b, 1, hq // h * t, -1)
    return _soft(scores, visible, value).reshape(b, hq, t, d).to(q.dtype)


def _plain_selected(state):
    q, table, starts, chosen = state["query"], state["table"], state["starts"], state["selected"]
    b, hq, t, d = q.shape
    h, k = chosen.shape[1], chosen.shape[3]
    page = table[:, None, None].expand(b, h, t, -1).gather(3, chosen.clamp(min=0).long())
    head = torch.arange(h, device="cuda")[None, :, None, None]
    key, value = (x.flatten(3, 4) for x in _page_values(state["cache"], page.long(), head))  # [B, H, T, K * 64, D]
    i = torch.arange(t, device="cuda")[None, None, :, None]
    j = (chosen[..., None] * PAGE + torch.arange(PAGE, device="cuda")).flatten(3)
    visible = (j <= starts[:, None, None, None] + i) & (chosen >= 0).repeat_interleave(PAGE, 3) & (i < state["counts"][:, None, None, None])
    qs = (q.float() * d**-0.5).reshape(b, h, hq // h, t, d).transpose(2, 3)
    scores = torch.matmul(qs, key.transpose(-1, -2).contiguous())
    return _soft(scores, visible[:, :, :, None], value).transpose(2, 3).reshape(b, hq, t, d).to(q.dtype)


def _plain_select(state):
    q, table, starts, k = state["query"], state["table"], state["starts"], state["budget"]
    b, hq, t, d = q.shape
    held = table.clamp(min=0)
    bounds, scale = state["cache"]["bounds"][held].float(), state["cache"]["bound_scale"][held]  # [B, N, H, 2, D], [B, N, H]
    h, n = scale.shape[2], scale.shape[1]
    codes, q_scale = _quantise(q.float(), "int8")
    codes = codes.float()
    ends = torch.cat((codes.clamp(min=0), codes.clamp(max=0)), -1).reshape(b, h, hq // h * t, 2 * d)  # q+ meets the upper bound
    dots = torch.matmul(ends, bounds.permute(0, 2, 3, 4, 1).reshape(b, h, 2 * d, n).contiguous())  # whole numbers below 2^24
    score = (dots.view(b, h, hq // h, t, n) * q_scale.view(b, h, hq // h, t, 1)).amax(2) * scale.transpose(1, 2)[:, :, None]
    i = torch.arange(t, device="cuda")[None]
    own_page = ((starts[:, None] + i) // PAGE)[:, None, :, None]
    at = torch.arange(n, device="cuda")
    score = torch.where(at < own_page, score, -math.inf)
    order = score.sort(dim=-1, descending=True, stable=True).indices[..., : k - 1]
    order = torch.where(order < own_page, order, n)  # fewer earlier pages than asked for
    order = torch.cat((own_page.expand(b, h, t, 1), order), -1).sort(-1).values
    out = torch.full((b, h, t, k), -1, dtype=torch.int32, device="cuda")
    real = (i < state["counts"][:, None])[:, None, :, None]
    out[..., : order.shape[-1]] = torch.where((order < n) & real, order, -1)
    return out


# ---- what a pass cannot do without ------------------------------------------------------------------------------------


def work(case):
    """Of a ragged case: with the middle of each range in the place of its lengths."""
    b, hq, h, d, k = (case[x] for x in ("batch", "heads", "kv_heads", "d", "budget"))
    half = case["ragged"] and b > 1
    t = (1 + case["tokens"]) / 2 if half else case["tokens"]
    context = 0.625 * case["context"] if half else case["context"]
    token = 2 * (d + 4)  # codes and scales of K and V of a token and head
    io = 2 * 2 * d * hq * t * b  # query and output
    if case["op"] == "read":
        return {"bytes": b * h * (t * token + case["tokens"] * 4 * d), "flops": 2 * b * h * t * d}
    if case["op"] == "write":  # read in 16 bits, written in 8, read back
        return {"bytes": b * h * (t * (4 * d + 2 * token) + case["tokens"] * 4 * d), "flops": 8 * b * h * t * d}
    if case["op"] == "select":
        pages = (context + t / 2) / PAGE
        return {"bytes": b * h * pages * (2 * d + 4) + io / 2 + 4 * b * h * case["tokens"] * k, "flops": 4 * b * hq * t * pages * d}
    if case["op"] == "selected":
        keys = PAGE * min(k, (context + t / 2) / PAGE + 1)
        # pages that several tokens of a sequence select are read once
        return {"bytes": b * h * min(t * keys, context + t) * token + io + 4 * b * h * t * k, "flops": 4 * b * hq * t * keys * d}
    pairs = t * (context + (t + 1) / 2)
    return {"bytes": b * h * (context + t) * token + io, "flops": 4 * b * hq * pairs * d}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------


def _exact_values(cache, name, d):
    """All of a cache's keys or values [P, H, 64, D] in FP64."""
    x = cache[name].double()
    if name == "value":
        x = torch.stack([x[..., j] for j in range(8)], 3).reshape(*x.shape[:2], PAGE, d)
    return x * cache[name + "_scale"].double().unsqueeze(-1)


def _exact_codes(x, codes):
    """What the quantiser makes of FP64 rows, as the values that it stands for."""
    largest = _CODES[codes][1]
    a = x.abs().max(-1, keepdim=True).values
    y = x * (largest / a)
    if codes == "int8":
        y = y.round()
    else:  # four significant bits, multiples of 2^-9 below 2^-6
        step = torch.exp2((torch.frexp(y)[1] - 1).clamp(min=-6).double() - 3)
        y = (y / step).round() * step
    return torch.where(a < _TINY, 0.0, y * (a / largest))


def exact(case, seed):
    if case["op"] == "select":
        return None  # whole numbers
    state = prepare(case, seed)
    b, h, d, t = case["batch"], case["kv_heads"], case["d"], case["tokens"]
    starts, counts, table = state["starts"].tolist(), state["counts"].tolist(), state["table"].long()
    if case["op"] == "write":
        out = {}
        for name in ("key", "value"):
            out[name] = torch.zeros((b, h, t, d), dtype=torch.float64, device="cuda")
            for r in range(b):
                out[name][r, :, : counts[r]] = _exact_codes(state[name][r, :, : counts[r]].double(), case["codes"])
        return {**out, "bounds": None, "bound_scale": None}
    cache = state["cache"]
    if case["op"] == "read":
        out = {n: torch.zeros((b, h, t, d), dtype=torch.float64, device="cuda") for n in ("key", "value")}
    else:
        q, hq = state["query"].double(), case["heads"]
        out = torch.zeros((b, hq, t, d), dtype=torch.float64, device="cuda")
    for r in range(b):
        pages = table[r, : (starts[r] + counts[r] + PAGE - 1) // PAGE]
        own_pages = {n: x[pages] for n, x in cache.items()}
        total = starts[r] + counts[r]
        kd, vd = (_exact_values(own_pages, n, d).permute(1, 0, 2, 3).reshape(h, -1, d)[:, :total] for n in ("key", "value"))
        if case["op"] == "read":
            out["key"][r, :, : counts[r]], out["value"][r, :, : counts[r]] = kd[:, starts[r] :], vd[:, starts[r] :]
            continue
        at = torch.arange(total, device="cuda")
        rows = torch.arange(counts[r], device="cuda")
        sees = at[None] <= starts[r] + rows[:, None]
        if case["op"] == "tree":
            sees = torch.cat((torch.ones((counts[r], starts[r]), dtype=torch.bool, device="cuda"), state["mask"][r, : counts[r], : counts[r]]), 1)
        group = hq // h
        step = max(1, (1 << 27) // total)  # 1 GiB of scores at a time
        for head in range(hq):
            kt, v = kd[head // group].t().contiguous(), vd[head // group]
            for i in range(0, counts[r], step):
                allowed = sees[i : i + step]
                if case["op"] == "selected":
                    listed_pages = state["selected"][r, head // group, i : min(i + step, counts[r])].long()
                    has = torch.zeros((listed_pages.shape[0], pages.numel() + 1), dtype=torch.bool, device="cuda")
                    has.scatter_(1, torch.where(listed_pages < 0, pages.numel(), listed_pages), True)
                    allowed = allowed & has[:, :-1].repeat_interleave(PAGE, 1)[:, :total]
                s = torch.mm(q[r, head, i : min(i + step, counts[r])], kt) * d**-0.5
                s = torch.where(allowed, s, -math.inf)
                p = torch.exp(s - s.max(1, keepdim=True).values)
                out[r, head, i : min(i + step, counts[r])] = torch.mm(p, v) / p.sum(1, keepdim=True)
    return out
