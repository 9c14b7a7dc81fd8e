"""Plain 64-bit statement of the 8-bit block-scaled cache (append, attention, evict) on CPU tensors, token by token."""

from __future__ import annotations

import math

import torch

TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def needed_scale(amax: float, dtype) -> float:
    if amax == 0:
        return 1.0
    e = -100
    while amax > TOP[dtype] * 2.0 ** e:
        e += 1
    return 2.0 ** e


def rounded(x: torch.Tensor, dtype) -> torch.Tensor:
    """float64 values in the codes' range -> the nearest codes (ties to even), as float64."""
    x = torch.where(torch.isnan(x), torch.zeros_like(x), x).clamp(-TOP[dtype], TOP[dtype])
    if dtype == torch.int8:
        return torch.round(x)
    _, exponent = torch.frexp(x)                       # |x| in [2^(exponent - 1), 2^exponent)
    step = torch.ldexp(torch.ones_like(x), (exponent - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def raw(x: torch.Tensor, dtype) -> torch.Tensor:
    """Code values -> the cache's bytes."""
    return x.to(torch.int8).view(torch.uint8) if dtype == torch.int8 else x.to(torch.float8_e4m3fn).view(torch.uint8)


class Cache:
    """CPU copy of a cache: `value` float64 code values, `byte` their bytes, `scale` float64, `weight` float64."""

    def __init__(self, codes, scales, weights=None):
        self.dtype = codes.dtype
        codes = codes.detach().cpu()
        self.byte = codes.view(torch.uint8).clone()
        self.value = codes.to(torch.float32).double()
        self.scale = scales.detach().cpu().double()
        self.weight = weights.detach().cpu().double() if weights is not None else None
        self.page = codes.shape[3]

    def put(self, plane, block, head, slot, value):
        self.value[plane, block, head, slot] = value
        self.byte[plane, block, head, slot] = raw(value, self.dtype)

    def append(self, key, value, starts, lengths, table):
        blocks, heads = self.value.shape[1:3]
        for r, length in enumerate(lengths):
            rows = list(range(starts[r], starts[r + 1]))
            first = length - len(rows)
            by_block = {}
            for i, row in enumerate(rows):
                if first + i >= 0 and (first + i) // self.page < len(table[r]):
                    by_block.setdefault((first + i) // self.page, []).append((row, (first + i) % self.page))
            for b, members in by_block.items():
                block = int(table[r][b])
                if not 0 <= block < blocks:
                    continue
                old = max(0, first) - b * self.page
                for plane, source in enumerate((key, value)):
                    for head in range(heads):
                        x = torch.stack([source[row, head].detach().cpu().double() for row, _ in members])
                        finite = x.abs()[torch.isfinite(x)]
                        amax = float(finite.max()) if finite.numel() else 0.0
                        scale = needed_scale(amax, self.dtype)
                        if old > 0:
                            before = float(self.scale[plane, block, head])
                            scale = max(scale, before) if amax > 0 else before
                            if scale > before:
                                for slot in range(old):
                                    again = rounded(self.value[plane, block, head, slot] * (before / scale), self.dtype)
                                    self.put(plane, block, head, slot, again)
                        for (_, slot), one in zip(members, x):
                            self.put(plane, block, head, slot, rounded(one / scale, self.dtype))
                            if self.weight is not None:
                                self.weight[block, head, slot] = 0.0
                        self.scale[plane, block, head] = scale

    def cached(self, plane, head, row_table, n):
        """The request's first n cached values of a head; the positions in blocks outside the cache are left out."""
        at = [(int(row_table[t // self.page]), t % self.page) for t in range(min(n, len(row_table) * self.page))]
        places = [(b, s) for b, s in at if 0 <= b < self.value.shape[1]]
        if not places:
            return torch.zeros(0, self.value.shape[4], dtype=torch.float64), places
        b, s = torch.tensor([p[0] for p in places]), torch.tensor([p[1] for p in places])
        return self.value[plane, b, head, s] * self.scale[plane, b, head][:, None], places

    def attention(self, query, starts, lengths, table, scale, accumulate=False, limit=None):
        """(output, lse, how far each may be off per unit: see `tolerance`) for the batch's real rows."""
        query = query.detach().cpu().double()
        heads, dim = query.shape[1:]
        group = heads // self.value.shape[2]
        out = torch.zeros_like(query)
        lse = torch.full(query.shape[:2], -math.inf, dtype=torch.float64)
        magnitude, spread = torch.zeros_like(query), torch.zeros(query.shape[:2], dtype=torch.float64)
        added = torch.zeros_like(self.weight) if accumulate else None
        for r, length in enumerate(lengths):
            count = starts[r + 1] - starts[r]
            for h in range(heads):
                end = max(0, length) if limit is None else min(max(0, length), limit)
                keys, places = self.cached(0, h // group, table[r], end)
                values, _ = self.cached(1, h // group, table[r], end)
                order = [t for t in range(min(end, len(table[r]) * self.page)) if 0 <= int(table[r][t // self.page]) < self.value.shape[1]]
                for i in range(count):
                    row = starts[r] + i
                    n = sum(1 for t in order if t <= length - count + i)
                    if n == 0:
                        continue
                    s = keys[:n] @ query[row, h] * scale
                    w = torch.softmax(s, 0)
                    lse[row, h] = torch.logsumexp(s, 0)
                    out[row, h] = w @ values[:n]
                    magnitude[row, h] = w @ values[:n].abs()
                    spread[row, h] = float((keys[:n].abs() @ query[row, h].abs()).max()) * scale
                    if accumulate:
                        for (b, slot), x in zip(places[:n], w.tolist()):
                            added[b, h // group, slot] += x
        return out, lse, magnitude, spread, added

    def evict(self, lengths, table, budget, sinks, recent):
        heads = self.value.shape[2]
        kept = torch.full((len(lengths), heads, budget), -1, dtype=torch.int32)
        left = torch.tensor([min(max(n, 0), budget) for n in lengths], dtype=torch.int32)
        for r, n in enumerate(lengths):
            for head in range(heads):
                if n <= budget:
                    kept[r, head, :max(n, 0)] = torch.arange(max(n, 0))
                    continue
                place = [(int(table[r][t // self.page]), t % self.page) for t in range(n)]
                weight = [float(self.weight[b, head, s]) for b, s in place]
                middle = sorted(range(sinks, n - recent), key=lambda t: (-weight[t] if weight[t] == weight[t] else math.inf, t))
                mine = sorted(list(range(sinks)) + list(range(n - recent, n)) + middle[:budget - sinks - recent])
                kept[r, head] = torch.tensor(mine)
                moved = [[self.value[plane, place[t][0], head, place[t][1]] * self.scale[plane, place[t][0], head] for t in mine]
                         for plane in range(2)]
                for b in range(0, budget, self.page):
                    block = int(table[r][b // self.page])
                    for plane in range(2):
                        x = torch.stack(moved[plane][b:b + self.page])
                        scale = needed_scale(float(x.abs().max()), self.dtype)
                        for slot, one in enumerate(x):
                            self.put(plane, block, head, slot, rounded(one / scale, self.dtype))
                        self.scale[plane, block, head] = scale
                    for slot, t in enumerate(mine[b:b + self.page]):
                        self.weight[block, head, slot] = weight[t]
        return kept, left


def tolerance(out, magnitude, spread, tokens, dtype, top):
    """How far an output may be from the 64-bit one: half a step of its type; fp16 softmax weights (half a step, 2^-12 of each
    relative to its own binade's top, 2^-11 at most, plus the smallest fp16 step 2^-24 halved, 2^-7 below the largest weight,
    for each token); scores and sums in fp32: a score of terms adding up to `spread` in magnitude is off by at most
    head_dim + 8 roundings of 2^-24, and twice that is what its weight relative to the others moves by."""
    dim = out.shape[-1]
    score = (2 * (dim + 8) * 2.0 ** -24 * spread + 2.0 ** -18)[..., None]
    return (torch.finfo(dtype).eps / 2 * out.abs() + (2.0 ** -11 + score) * magnitude * (1 + 2.0 ** -8)
            + tokens * 2.0 ** -32 * top + torch.finfo(dtype).tiny)
