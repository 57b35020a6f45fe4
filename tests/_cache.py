"""The quantised cache's definition on the CPU, for its tests: codes, scales, bounds and selections exactly (every step
is one FP32 operation or a whole number), attention in FP64 with a bound of the kernel's rounding."""

from __future__ import annotations

import math

import torch

PAGE = 64
LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
TINY = 2.0**-118


def quantise(x: torch.Tensor, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of rows [..., D], by the rule of ``include/piper_cache.h``."""
    x = x.float()
    finite = torch.isfinite(x).all(-1, keepdim=True)
    safe = torch.where(finite, x, 0.0)
    a = safe.abs().amax(-1, keepdim=True)
    top = torch.full((), LARGEST[dtype])
    zero = a < TINY
    y = safe * torch.where(zero, 0.0, top / torch.where(zero, top, a))
    if dtype is torch.int8:
        y = y.round()
    codes = y.clamp(-top, top).to(dtype)
    scale = torch.where(finite, torch.where(zero, 0.0, a / top), math.nan)
    return codes, scale.squeeze(-1)


class Model:
    """A cache's arrays on the CPU, written token by token; ``fill`` starts it with arbitrary bytes."""

    def __init__(self, pages: int, heads: int, d: int, dtype: torch.dtype, fill: int | None = None):
        self.shape, self.dtype = (pages, heads, d), dtype
        if fill is None:
            codes = lambda *s: torch.zeros(s, dtype=torch.int8)  # noqa: E731
            floats = lambda *s: torch.zeros(s)  # noqa: E731
        else:
            g = torch.Generator().manual_seed(fill)
            codes = lambda *s: torch.randint(-128, 128, s, generator=g, dtype=torch.int8)  # noqa: E731
            floats = lambda *s: torch.where(torch.rand(s, generator=g) < 0.3, math.nan, torch.randn(s, generator=g))  # noqa: E731
        self.key = codes(pages, heads, PAGE, d).view(dtype)
        self.key_scale = floats(pages, heads, PAGE)
        self.value = codes(pages, heads, 8, d, 8).view(dtype)
        self.value_scale = floats(pages, heads, PAGE)
        self.bounds = codes(pages, heads, 2, d)
        self.bound_scale = floats(pages, heads)

    def arrays(self) -> tuple[torch.Tensor, ...]:
        return (self.key, self.key_scale, self.value, self.value_scale, self.bounds, self.bound_scale)

    def page_of(self, table, b: int, position: int) -> int:
        if position < 0 or position // PAGE >= table.shape[1]:
            return -1
        p = int(table[b, position // PAGE])
        return p if 0 <= p < self.shape[0] else -1

    def write(self, key, value, table, starts, counts=None) -> None:
        batch, _, tokens, _ = key.shape
        kc, ks = quantise(key, self.dtype)
        vc, vs = quantise(value, self.dtype)
        full = set()
        for b in range(batch):
            count = tokens if counts is None else max(0, min(tokens, int(counts[b])))
            for i in range(count):
                position = int(starts[b]) + i
                page, slot = self.page_of(table, b, position), position % PAGE
                if page < 0:
                    continue
                self.key.view(torch.int8)[page, :, slot] = kc[b, :, i].view(torch.int8)
                self.key_scale[page, :, slot] = ks[b, :, i]
                self.value.view(torch.int8)[page, :, slot // 8, :, slot % 8] = vc[b, :, i].view(torch.int8)
                self.value_scale[page, :, slot] = vs[b, :, i]
                if slot == PAGE - 1:
                    full.add(page)
        for page in full:
            k = self.key[page].float() * self.key_scale[page][..., None]  # [H, 64, D]
            bad = k.isnan()
            upper = torch.where(bad, -math.inf, k).amax(1)
            lower = torch.where(bad, math.inf, k).amin(1)
            none = upper < lower
            ends = torch.stack((torch.where(none, 0.0, upper), torch.where(none, 0.0, lower)), 1)  # [H, 2, D]
            codes, scale = quantise(ends.flatten(1), torch.int8)
            self.bounds[page] = codes.view(ends.shape)
            self.bound_scale[page] = scale

    def tokens(self, table, b: int, positions) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """FP32 keys and values [H, n, D] of positions, and which of them have a page; zeros where not."""
        _, h, d = self.shape
        pages = torch.tensor([self.page_of(table, b, int(p)) for p in positions], dtype=torch.long)
        slots = torch.tensor([int(p) % PAGE for p in positions], dtype=torch.long)
        there = pages >= 0
        page = pages.clamp(min=0)
        k = self.key.view(torch.int8)[page, :, slots].view(self.dtype).float() * self.key_scale[page, :, slots][..., None]
        v = self.value.view(torch.int8)[page, :, slots // 8, :, slots % 8].contiguous().view(self.dtype).float()
        v = v * self.value_scale[page, :, slots][..., None]
        return (torch.where(there[:, None, None], k, 0.0).transpose(0, 1), torch.where(there[:, None, None], v, 0.0).transpose(0, 1), there)

    def read(self, table, starts, counts, size: int, dtype: torch.dtype):
        _, h, d = self.shape
        out = torch.zeros((2, table.shape[0], h, size, d), dtype=dtype)
        for b in range(table.shape[0]):
            count = size if counts is None else max(0, min(size, int(counts[b])))
            if count:
                k, v, _ = self.tokens(table, b, range(int(starts[b]), int(starts[b]) + count))
                out[0, b, :, :count], out[1, b, :, :count] = k.to(dtype), v.to(dtype)
        return out[0], out[1]

    def attention(self, q, table, starts, counts=None, mask=None, selected=None, scale=None):
        """FP64 output and, per value, how far a kernel's may be from it: half a step of the output type; P rounded
        to a 16-bit float of 11 bits (2^-11 of the sum of p |v|); score errors of FP32 sums of D products, which change
        each p by twice their size relatively; an FP32 exp2 and the sums (2^-18 of the sum of p |v|).  Where a key's weight
        is below 2^-29 of the largest, its 16-bit P is a subnormal: with w = p s 2^15 / r, s the key's value scale and r < 2 s'
        for the largest value scale s' of the pages, w is off by at most 2^-25, the key's part w c r / 2^15 (|c| <= L) by
        2^-25 r L / 2^15 < 2^-39 s' L: 2^-39 of the largest value a page of the K/V head holds, for each key seen."""
        batch, heads, tokens, d = q.shape
        _, h, _ = self.shape
        scale = d**-0.5 if scale is None else scale
        out = torch.zeros(q.shape, dtype=torch.float64)
        spread = torch.zeros(q.shape, dtype=torch.float64)
        for b in range(batch):
            count = tokens if counts is None else max(0, min(tokens, int(counts[b])))
            start = int(starts[b])
            n = min(start + count, table.shape[1] * PAGE)
            if count == 0 or n <= 0:
                continue
            k, v, there = (x.double() if x.dtype is not torch.bool else x for x in self.tokens(table, b, range(n)))
            at = torch.arange(n)
            largest = v.nan_to_num(nan=0.0).abs().amax((1, 2))  # per K/V head, seen by the row or not
            for i in range(count):
                if mask is None:
                    sees = at <= start + i
                else:
                    row = mask[b % mask.shape[0], i]
                    sees = (at < start) | ((at >= start) & row[(at - start).clamp(0, tokens - 1)])
                times = (sees & there).double()[None].expand(h, n)
                if selected is not None:
                    named = torch.zeros((h, n // PAGE + 2), dtype=torch.float64)
                    for kv in range(h):
                        for p in selected[b, kv, i].tolist():
                            if 0 <= p < named.shape[1]:
                                named[kv, p] += 1
                    times = times * named.repeat_interleave(PAGE, 1)[:, :n]
                for head in range(heads):
                    kv = head // (heads // h)
                    use = times[kv] > 0
                    if not bool(use.any()):
                        continue
                    qs = q[b, head, i].double()
                    s = (k[kv][use] @ qs) * scale
                    p = times[kv][use] * torch.exp(s - s.max())
                    total = p.sum()
                    out[b, head, i] = (p @ v[kv][use]) / total
                    size = float((k[kv][use].abs() @ qs.abs()).max()) * scale
                    e = 2 * size * (d + 4) * 2.0**-24
                    spread[b, head, i] = (2.0**-11 + 2.0**-18 + e) * (p @ v[kv][use].abs()) / total + float(use.sum()) * 2.0**-39 * largest[kv]
        bound = spread + out.abs() * torch.finfo(q.dtype).eps / 2 + (2.0**-25 if q.dtype is torch.float16 else 0.0)
        return out, bound

    def select(self, q, table, starts, counts, budget: int) -> torch.Tensor:
        batch, heads, tokens, d = q.shape
        pages, h, _ = self.shape
        codes, scales = quantise(q, torch.int8)
        codes = codes.long()
        out = torch.full((batch, h, tokens, budget), -1, dtype=torch.int32)
        for b in range(batch):
            count = tokens if counts is None else max(0, min(tokens, int(counts[b])))
            for i in range(count):
                position = int(starts[b]) + i
                if position < 0 or position >= table.shape[1] * PAGE:
                    continue
                own = position // PAGE
                named = table[b, :own].long()
                ok = (named >= 0) & (named < pages)
                held = torch.where(ok, named, 0)
                for kv in range(h):
                    bounds, bscale = self.bounds[held, kv].long(), self.bound_scale[held, kv]
                    score = None
                    for head in range(kv * (heads // h), (kv + 1) * (heads // h)):
                        c = codes[b, head, i]
                        dot = (c.clamp(min=0) * bounds[:, 0] + c.clamp(max=0) * bounds[:, 1]).sum(-1).float() * scales[b, head, i]
                        score = dot if score is None else torch.fmax(score, dot)
                    score = torch.where(ok, score * bscale, -math.inf).nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf)
                    best = score.sort(descending=True, stable=True).indices[: budget - 1]
                    chosen = sorted(best.tolist() + [own])
                    out[b, kv, i, : len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
        return out


def table_of(widths: list[int], pages: int, seed: int) -> torch.Tensor:
    """Distinct pages in no order for sequences of ``widths`` pages; -1 behind them."""
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g).int()
    table = torch.full((len(widths), max(widths)), -1, dtype=torch.int32)
    at = 0
    for b, w in enumerate(widths):
        table[b, :w] = order[at : at + w]
        at += w
    assert at <= pages
    return table


def tokens_of(b: int, h: int, t: int, d: int, dtype: torch.dtype, seed: int, layout: str = "bhtd") -> torch.Tensor:
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((b, h, t, d), generator=g) + torch.randn((1, h, 1, d), generator=g)
    x = (x * torch.exp(0.5 * torch.randn((b, h, t, 1), generator=g))).to(dtype)
    if layout == "bthd":
        return x.transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "odd":  # rows at odd multiples of two bytes: copied by the operators
        return torch.cat([x, x[..., :1]], -1)[..., :d]
    return x


def tree_mask(b: int, t: int, seed: int) -> torch.Tensor:
    """Each node sees itself and its ancestors; a node's parent stands before it."""
    g = torch.Generator().manual_seed(seed)
    mask = torch.zeros((b, t, t), dtype=torch.bool)
    for r in range(b):
        for i in range(t):
            if i:
                mask[r, i] = mask[r, int(torch.randint(max(0, i - 5), i, (1,), generator=g))]
            mask[r, i, i] = True
    return mask
