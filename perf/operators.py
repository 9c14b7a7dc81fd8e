"""Cases, plain forms and 64-bit values of the operators of an 8-bit block-scaled KV cache.

The cache holds K and V as 8-bit codes [2, blocks, kv heads, page tokens, channels] (e4m3 or int8) with one fp32 scale for each
(plane, block, kv head), and, where tokens are to be evicted, one fp32 accumulated attention weight for each (block, kv head,
token).  Three operators work on it:

  append     quantizes the K/V rows of a step's new tokens into their blocks.  A block's scale is the smallest power of two that
             brings its largest finite magnitude into the type's range (448 or 127); it only grows while a block fills up, and the
             block's earlier tokens are rounded again when it does.
  attention  softmax attention of each request's last rows over its cached tokens, causal among these rows; optionally adds every
             token's weight, summed over rows and the query heads of its kv head, to the accumulated weights.
  evict      keeps, for each request and kv head, the first `sinks` tokens, the last `recent` ones and those of the others that have
             the largest accumulated weight (ties: the lowest position), `budget` in all; moves them to the front of the request's
             blocks in their order, and gives each block the scale that its tokens need.

Codes are returned in their own type (float8_e4m3fn or int8) beside the scales: both are determined to the bit.
"""

import math
import random

import torch

own = False

TOP = {"fp8": 448.0, "int8": 127.0}
TYPE = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}
ACTIVATION = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---- cases -------------------------------------------------------------------------------------------------------------

def listed():
    base = {"page": 16, "kind": "fp8", "act": "bf16", "rows": 1, "pad": 0, "weights": False, "mix": 1}
    attention = dict(base, op="attention")
    append = dict(base, op="append")
    evict = dict(base, op="evict", weights=True)
    return [
        # the next token of one short conversation: only latency counts
        dict(attention, name="attention 1x97", requests=1, lo=97, hi=97, heads=16, kv_heads=16, dim=128),
        # a full batch of looped-decoder heads at the benchmark's shape: 64 sequences of 8192 tokens
        dict(attention, name="attention 64x8192", requests=64, lo=8192, hi=8192, heads=16, kv_heads=16, dim=128),
        # a mixed batch in service, shared KV heads, int8 codes, large pages, a few padded rows behind the last sequence
        dict(attention, name="attention ragged int8", requests=40, lo=1, hi=16001, heads=32, kv_heads=8, dim=128,
             kind="int8", page=32, pad=8, mix=2),
        # one very long document
        dict(attention, name="attention 1x131071", requests=1, lo=131071, hi=131071, heads=32, kv_heads=4, dim=128, act="fp16"),
        # drafted tokens are verified: up to 5 rows a request, an odd head count of narrow heads
        dict(attention, name="attention verify d96", requests=16, lo=700, hi=5003, heads=55, kv_heads=55, dim=96, rows=5, mix=3),
        # decode that keeps track of what is attended to
        dict(attention, name="attention + weights", requests=32, lo=4100, hi=4100, heads=32, kv_heads=8, dim=128, weights=True),
        # one step's new tokens of a batch
        dict(append, name="append 64 tokens", requests=64, lo=1, hi=8000, heads=16, kv_heads=16, dim=128, mix=4),
        # prompts of a step, most of them new, in ragged lengths
        dict(append, name="append prompts", requests=12, lo=0, hi=300, heads=16, kv_heads=16, dim=128, rows=4001, kind="int8", mix=5),
        # a batch whose sequences have outgrown their budget
        dict(evict, name="evict 32 to 2048", requests=32, lo=4097, hi=9001, heads=16, kv_heads=16, dim=128, budget=2048, sinks=4,
             recent=256, mix=6),
        # a few short ones
        dict(evict, name="evict 3 to 111", requests=3, lo=130, hi=401, heads=7, kv_heads=7, dim=64, budget=111, sinks=1, recent=30,
             kind="int8", mix=7),
        # one long document is brought down to an eighth
        dict(evict, name="evict 131071 to 16384", requests=1, lo=131071, hi=131071, heads=32, kv_heads=8, dim=128, budget=16384,
             sinks=16, recent=1024, kind="int8", page=32),
    ]


def _between(rng, lo, hi):
    """A whole number spread over lo..hi on a logarithmic scale."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "append", "evict"])
    case = {"op": op, "page": rng.choice([16, 32]), "kind": rng.choice(["fp8", "int8"]), "act": rng.choice(["bf16", "fp16"]),
            "dim": rng.choice([64, 96, 128, 128]), "rows": 1, "pad": 0, "weights": op == "evict", "mix": rng.randrange(1 << 20)}
    case["kv_heads"] = rng.choice([1, 2, 3, 4, 7, 8, 11, 16])
    case["heads"] = case["kv_heads"] * rng.choice([1, 1, 2, 4, 5, 8])
    most = (1 << 28) // (case["kv_heads"] * case["dim"])  # cached tokens, padded to the longest sequence
    if op == "attention":
        case["rows"] = rng.choice([1, 1, 1, 2, 4, 7, 33])
        case["weights"] = rng.random() < 0.3
        case["pad"] = rng.choice([0, 0, 5])
        most = min(most, (1 << 27) // (case["heads"] * case["rows"]))
        case["requests"] = _between(rng, 1, 96)
        case["hi"] = _between(rng, 1, max(1, min(131072, most // case["requests"])))
        case["lo"] = rng.choice([1, case["hi"], max(1, case["hi"] // 3)])
    elif op == "append":
        case["requests"] = _between(rng, 1, 200)
        case["rows"] = _between(rng, 1, max(1, min(8192, 40000 // case["requests"])))
        case["hi"] = _between(rng, 1, 2000)
        case["lo"] = rng.choice([0, case["hi"]])
        case["pad"] = rng.choice([0, 3])
    else:
        case["requests"] = _between(rng, 1, 48)
        case["hi"] = _between(rng, 40, max(64, min(131072, most // case["requests"])))
        case["lo"] = max(1, case["hi"] // rng.choice([1, 2, 10]))
        case["budget"] = _between(rng, 8, case["hi"])
        case["sinks"] = rng.randrange(0, 1 + case["budget"] // 4)
        case["recent"] = rng.randrange(0, 1 + case["budget"] // 2)
    return case


def shape(case):
    """(rows of each request, cached tokens of each request, the new ones included).  For `append`, lo..hi counts the tokens that
    were there before."""
    rng = random.Random(case["mix"])
    rows = [case["rows"]] + [rng.randint(max(1, case["rows"] // 2), case["rows"]) for _ in range(case["requests"] - 1)]
    spread = [case["hi"]]
    for _ in range(case["requests"] - 1):
        spread.append(_between(rng, case["lo"], case["hi"]) if case["lo"] else rng.choice([0, 0, rng.randint(1, case["hi"])]))
    if case["op"] == "append":
        return rows, [old + new for old, new in zip(spread, rows)]
    return rows, [max(total, 1) for total in spread]


def work(case):
    rows, lengths = shape(case)
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    pages = sum(-(-n // case["page"]) for n in lengths)
    if case["op"] == "attention":
        seen = sum(max(0, n - q + i + 1) for n, q in zip(lengths, rows) for i in range(q))
        size = sum(lengths) * kv * 2 * dim + pages * (4 + kv * 8) + sum(rows) * heads * (4 * dim + 4)
        if case["weights"]:
            size += sum(lengths) * kv * 8
        return {"bytes": size, "flops": 4 * dim * heads * seen}
    if case["op"] == "append":
        new = sum(rows) * kv * 2 * dim
        touched = sum((n - 1) // case["page"] - (n - q) // case["page"] + 1 for n, q in zip(lengths, rows))
        return {"bytes": 3 * new + touched * kv * 2 * 4, "flops": 3 * new}
    gone = [n for n in lengths if n > case["budget"]]
    size = sum(n * 4 + case["budget"] * (4 * dim + 8) for n in gone) * kv + case["requests"] * kv * case["budget"] * 4
    return {"bytes": size, "flops": sum(n + 4 * case["budget"] * dim for n in gone) * kv}


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def prepare(case, seed):
    device = _device()
    make = torch.Generator(device=device).manual_seed(seed)
    rows, lengths = shape(case)
    page, kv, dim, act = case["page"], case["kv_heads"], case["dim"], ACTIVATION[case["act"]]
    counts = [-(-n // page) for n in lengths]
    blocks = sum(counts) + 3
    # block 0 is the null block: it fills the table behind a sequence's pages
    order = 1 + torch.randperm(blocks - 1, generator=make, device=device)
    table = torch.zeros(len(rows), max(counts) + 1, dtype=torch.int32, device=device)
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = order[at:at + n]
        at += n
    # keys have a few strong channels, as rotary keys do; blocks differ in magnitude
    spread = torch.ones(2, kv, 1, dim, device=device)
    spread[0] += 3.0 * (torch.rand(kv, 1, dim, generator=make, device=device) > 0.95)
    codes = torch.empty(2, blocks, kv, page, dim, dtype=TYPE[case["kind"]], device=device)
    scales = torch.empty(2, blocks, kv, device=device)
    step = max(1, (1 << 26) // (kv * page * dim))
    for plane in range(2):
        for b in range(0, blocks, step):
            n = min(step, blocks - b)
            x = torch.randn(n, kv, page, dim, generator=make, device=device) * spread[plane]
            x *= 0.5 + torch.rand(n, kv, 1, 1, generator=make, device=device)
            scale = _needed_scale(x.abs().amax((2, 3)), case["kind"])
            codes[plane, b:b + n] = _encode(x / scale[..., None, None], case["kind"])
            scales[plane, b:b + n] = scale
    total = sum(rows) + case["pad"]
    state = {"op": case["op"], "kind": case["kind"], "codes": codes, "scales": scales, "weights": None, "table": table,
             "starts": torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], dtype=torch.int32, device=device),
             "lengths": torch.tensor(lengths, dtype=torch.int32, device=device), "most_rows": max(rows), "longest": max(lengths)}
    if case["weights"]:
        # accumulated weights are heavy-tailed, and many tokens were hardly looked at
        w = torch.exp(2.0 * torch.randn(blocks, kv, page, generator=make, device=device))
        state["weights"] = torch.where(torch.rand(w.shape, generator=make, device=device) < 0.1, torch.zeros_like(w), w)
    if case["op"] == "attention":
        state["query"] = (1.5 * torch.randn(total, case["heads"], dim, generator=make, device=device)).to(act)
        state["out"] = torch.zeros_like(state["query"])
        state["lse"] = torch.zeros(total, case["heads"], device=device)
    elif case["op"] == "append":
        x = torch.randn(2, total, kv, dim, generator=make, device=device) * spread[:, None, :, 0]
        x *= 0.5 + 1.5 * torch.rand(2, total, kv, 1, generator=make, device=device)
        state["key"], state["value"] = x[0].to(act), x[1].to(act)
    else:
        state.update(budget=case["budget"], sinks=case["sinks"], recent=case["recent"],
                     kept=torch.full((len(rows), kv, case["budget"]), -1, dtype=torch.int32, device=device),
                     left=torch.zeros(len(rows), dtype=torch.int32, device=device))
    if own:
        from residualquant_b200.block_cache import BlockCache

        state["cache"] = BlockCache(codes, scales, state["weights"])
    return state


# ---- the framework's calls and the plain forms -----------------------------------------------------------------------------

def run(state):
    if state["op"] == "attention":
        if own:
            state["cache"].attention(state["query"], state["out"], state["starts"], state["lengths"], state["table"],
                                     lse=state["lse"], accumulate=state["weights"] is not None)
        else:
            _plain_attention(state)
        return [state["out"], state["lse"]] + ([state["weights"]] if state["weights"] is not None else [])
    if state["op"] == "append":
        if own:
            state["cache"].append(state["key"], state["value"], state["starts"], state["lengths"], state["table"])
        else:
            _plain_append(state)
        return [state["codes"], state["scales"]]
    if own:
        state["cache"].evict(state["lengths"], state["table"], state["budget"], sinks=state["sinks"], recent=state["recent"],
                             kept=state["kept"], new_lens=state["left"])
    else:
        _plain_evict(state)
    return [state["codes"], state["scales"], state["weights"], state["kept"], state["left"]]


def _needed_scale(amax, kind):
    """The smallest power of two that brings `amax` to at most the type's largest value; 1 for 0."""
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa * 2^exponent, mantissa in [0.5, 1)
    top, at = torch.frexp(torch.tensor(TOP[kind]))
    exponent = (exponent - int(at) + (mantissa > float(top)).to(exponent.dtype)).clamp(min=-100)
    power = ((exponent.to(torch.int32) + 127) << 23).view(torch.float32)  # exact, as a library's power need not be
    return torch.where(amax > 0, power, torch.ones_like(amax))


def _encode(x, kind):
    x = x.clamp(-TOP[kind], TOP[kind])
    return torch.round(x).to(torch.int8) if kind == "int8" else x.to(torch.float8_e4m3fn)


def _bytes(codes):
    return codes.view(torch.uint8)


def _rows_of(state):
    """Index of every request's rows [requests, most rows], whether it is one, and its position in the sequence."""
    starts, lengths = state["starts"].long(), state["lengths"].long()
    i = torch.arange(state["most_rows"], device=starts.device)
    count = starts[1:] - starts[:-1]
    return starts[:-1, None] + i, i < count[:, None], (lengths - count)[:, None] + i


def _plain_attention(state):
    codes, scales, table = state["codes"], state["scales"], state["table"].long()
    _, blocks, kv, page, dim = codes.shape
    index, real, position = _rows_of(state)
    requests, most = index.shape
    pages = -(-state["longest"] // page)
    table = table[:, :pages]
    query = state["query"]
    group = query.shape[1] // kv
    q = query[index.clamp(max=query.shape[0] - 1)].float().reshape(requests, most, kv, group, dim)
    q = q.permute(0, 2, 1, 3, 4).reshape(requests, kv, most * group, dim)

    def cached(plane):  # [requests, kv heads, tokens, channels]
        x = _bytes(codes[plane])[table].view(codes.dtype).float()
        x = x * scales[plane][table][..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(requests, kv, pages * page, dim)

    scores = (q @ cached(0).transpose(2, 3)) / math.sqrt(dim)
    token = torch.arange(pages * page, device=codes.device)
    seen = (token <= position[..., None]) & real[..., None]  # [requests, rows, tokens]
    seen = seen[:, None, :, None].expand(requests, kv, most, group, -1).reshape(scores.shape)
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, torch.zeros_like(p))
    o = (p @ cached(1)).reshape(requests, kv, most, group, dim).permute(0, 2, 1, 3, 4).reshape(requests, most, kv * group, dim)
    lse = (top + torch.log(total)).reshape(requests, kv, most, group).permute(0, 2, 1, 3).reshape(requests, most, kv * group)
    state["out"][index[real]] = o[real].to(query.dtype)
    state["lse"][index[real]] = lse[real]
    if state["weights"] is not None:
        added = p.sum(2).reshape(requests, kv, pages, page).permute(0, 2, 1, 3)  # nothing is added behind a sequence's end
        state["weights"].index_add_(0, table.reshape(-1), added.reshape(requests * pages, kv, page))


def _plain_append(state):
    codes, scales, table, kind = state["codes"], state["scales"], state["table"].long(), state["kind"]
    _, blocks, kv, page, dim = codes.shape
    index, real, position = _rows_of(state)
    request = torch.arange(index.shape[0], device=index.device)[:, None].expand_as(index)[real]
    row, at = index[real], position[real]
    block, slot = table[request, at // page], at % page
    first = at[state["starts"].long()[request]]  # the position of the request's first new token
    fresh = torch.zeros(blocks, dtype=torch.bool, device=row.device)
    fresh[block[slot == 0]] = True
    touched, where = torch.unique(block, return_inverse=True)
    before = torch.zeros(touched.numel(), dtype=torch.long, device=row.device)  # tokens that the block held before
    before[where] = (first - at + slot).clamp(min=0)
    before[fresh[touched]] = 0
    for plane, rows in enumerate((state["key"], state["value"])):
        x = rows[row].float()
        x = torch.where(torch.isnan(x), torch.zeros_like(x), x)
        size = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(2)
        amax = torch.zeros(touched.numel(), kv, device=x.device).index_reduce_(0, where, size, "amax")
        needed = _needed_scale(amax, kind)
        old = scales[plane][touched]
        needed = torch.where((before[:, None] > 0) & (amax == 0), old, needed)  # zeros fit any scale
        new = torch.where(before[:, None] > 0, torch.maximum(old, needed), needed)
        held = _bytes(codes[plane])[touched].view(codes.dtype)
        again = _encode(held.float() * (old / new)[..., None, None], kind)
        keep = torch.arange(page, device=x.device) < before[:, None]
        held = torch.where(keep[:, None, :, None], _bytes(again), _bytes(held))
        held[where, :, slot] = _bytes(_encode(x / new[where][..., None], kind))
        _bytes(codes[plane])[touched] = held
        scales[plane][touched] = new


def _plain_evict(state):
    codes, scales, weights, table, kind = state["codes"], state["scales"], state["weights"], state["table"].long(), state["kind"]
    _, blocks, kv, page, dim = codes.shape
    budget, sinks, recent = state["budget"], state["sinks"], state["recent"]
    n = state["lengths"].long()
    requests, pages = table.shape
    token = torch.arange(pages * page, device=codes.device)
    w = weights[table].permute(0, 2, 1, 3).reshape(requests, kv, pages * page)
    w = torch.where(torch.isnan(w), torch.full_like(w, -3e38), w)
    held = (token < sinks) | (token >= (n - recent)[:, None])
    w = torch.where(held[:, None], torch.full_like(w, math.inf), w)
    w = torch.where((token < n[:, None])[:, None], w, torch.full_like(w, -math.inf))
    kept = torch.sort(w, dim=2, descending=True, stable=True).indices[..., :budget].sort(2).values
    slots = torch.arange(min(budget, kept.shape[2]), device=codes.device)
    full = n > budget
    kept = torch.where(full[:, None, None], kept, slots.expand_as(kept))
    lasts = torch.minimum(n, torch.full_like(n, budget))
    alive = slots < lasts[:, None]  # [requests, budget]
    state["kept"].fill_(-1)
    state["kept"][..., :slots.numel()] = torch.where(alive[:, None], kept, torch.full_like(kept, -1)).to(torch.int32)
    state["left"].copy_(lasts)
    # the new blocks: the kept tokens, `page` at a time
    count = -(-slots.numel() // page)
    wide = torch.nn.functional.pad(kept, (0, count * page - slots.numel()))
    block = torch.gather(table[:, None].expand(requests, kv, pages), 2, wide // page)
    offset = wide % page
    head = torch.arange(kv, device=codes.device)[None, :, None]
    put = torch.nn.functional.pad(alive & full[:, None], (0, count * page - slots.numel()))
    put = put.reshape(requests, count, 1, page)
    target = table[:, :count]
    moved = weights[block, head, offset].reshape(requests, kv, count, page).transpose(1, 2)
    fresh = []
    for plane in range(2):
        x = _bytes(codes[plane])[block, head, offset].view(codes.dtype).float() * scales[plane][block, head][..., None]
        x = x.reshape(requests, kv, count, page, dim).transpose(1, 2)
        scale = _needed_scale(torch.where(put[..., None], x.abs(), torch.zeros_like(x)).amax((3, 4)), kind)
        fresh.append((_bytes(_encode(x / scale[..., None, None], kind)), scale))
    for plane, (code, scale) in enumerate(fresh):
        before = _bytes(codes[plane])[target]
        _bytes(codes[plane])[target] = torch.where(put[..., None], code, before)
        scales[plane][target] = torch.where(put.any(3), scale, scales[plane][target])
    weights[target] = torch.where(put, moved, weights[target])


# ---- 64 bits -----------------------------------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    return {"attention": _exact_attention, "append": _exact_append, "evict": _exact_evict}[case["op"]](case, state)




def _gathered(state, plane, ids):
    raw = state["codes"][plane].view(torch.uint8).index_select(0, ids).view(state["codes"].dtype).double()
    raw = raw * state["scales"][plane].index_select(0, ids).double().reshape(ids.numel(), -1, 1, 1)
    return raw.transpose(0, 1).flatten(1, 2)


def _exact_attention(case, state):
    rows, lengths = shape(case)
    kv, page, dim = case["kv_heads"], case["page"], case["dim"]
    group = case["heads"] // kv
    out = state["query"].double() * 0
    lse = out[..., 0].clone()
    weights = state["weights"].double() if state["weights"] is not None else None
    start = 0
    for r, (q, n) in enumerate(zip(rows, lengths)):
        ids = state["table"][r, :-(-n // page)].long()
        key, value = _gathered(state, 0, ids)[:, :n], _gathered(state, 1, ids)[:, :n]
        sums = torch.zeros(kv, ids.numel() * page, dtype=torch.float64, device=out.device)
        for i in range(q):
            see = n - q + i + 1
            if see <= 0:
                lse[start + i] = -math.inf
                continue
            one = state["query"][start + i].double().reshape(kv, group, dim)
            s = torch.einsum("hgd,htd->hgt", one, key[:, :see]) * dim ** -0.5
            lse[start + i] = torch.logsumexp(s, 2).flatten()
            p = torch.softmax(s, 2)
            out[start + i] = torch.einsum("hgt,htd->hgd", p, value[:, :see]).reshape(-1, dim)
            sums[:, :see] += p.sum(1)
        if weights is not None:
            weights[ids] += sums.reshape(kv, ids.numel(), page).transpose(0, 1)
        start += q
    return [out, lse] + ([weights] if weights is not None else [])


def _exact_scale(x, kind):
    """By the definition: the first power of two (from 2^-100 on) that times the type's largest value reaches the magnitude."""
    amax = x.abs().amax((-1, -2))
    powers = torch.tensor([2.0 ** e for e in range(-100, 128)], dtype=torch.float64, device=x.device)
    return torch.where(amax > 0, powers[torch.searchsorted(powers * TOP[kind], amax.contiguous())], torch.ones_like(amax))


def _exact_code(x, kind):
    if kind == "int8":
        return torch.round(x)
    # e4m3 has three bits behind the leading one, from 2^-6 up
    powers = torch.tensor([2.0 ** e for e in range(-6, 10)], dtype=torch.float64, device=x.device)
    step = powers[(torch.searchsorted(powers, x.abs().contiguous(), right=True) - 1).clamp(min=0)] / 8
    return torch.round(x / step) * step


def _exact_append(case, state):
    rows, lengths = shape(case)
    page, kind = case["page"], case["kind"]
    codes, scales = state["codes"].double(), state["scales"].double()
    table = state["table"].tolist()
    start = 0
    for r, (q, n) in enumerate(zip(rows, lengths)):
        for b in range((n - q) // page, (n - 1) // page + 1):
            first, last = max(b * page, n - q), min((b + 1) * page, n)
            for plane, source in enumerate((state["key"], state["value"])):
                x = source[start + first - (n - q):start + last - (n - q)].double().transpose(0, 1)
                scale, block, old = _exact_scale(x, kind), table[r][b], first - b * page
                if old:
                    zero = x.abs().amax((1, 2)) == 0
                    scale = torch.where(zero, scales[plane, block], torch.maximum(scale, scales[plane, block]))
                    was = codes[plane, block, :, :old] * (scales[plane, block] / scale)[:, None, None]
                    codes[plane, block, :, :old] = _exact_code(was, kind)
                codes[plane, block, :, old:old + last - first] = _exact_code(x / scale[:, None, None], kind)
                scales[plane, block] = scale
        start += q
    return [codes, scales]


def _exact_evict(case, state):
    _, lengths = shape(case)
    kv, page, kind, budget = case["kv_heads"], case["page"], case["kind"], case["budget"]
    codes, scales, weights = state["codes"].double(), state["scales"].double(), state["weights"].double()
    kept = torch.full((len(lengths), kv, budget), -1)
    for r, n in enumerate(lengths):
        kept[r, :, :min(n, budget)] = torch.arange(min(n, budget))
        if n <= budget:
            continue
        ids = state["table"][r, :-(-n // page)].long()
        target = ids[:-(-budget // page)]
        w = weights[ids].transpose(0, 1).flatten(1)[:, :n].cpu()
        free = budget - case["sinks"] - case["recent"]
        middle = w[:, case["sinks"]:n - case["recent"]]
        order = torch.argsort(middle, dim=1, descending=True, stable=True)[:, :free] + case["sinks"]
        ends = torch.cat([torch.arange(case["sinks"]), torch.arange(n - case["recent"], n)]).expand(kv, -1)
        mine = torch.cat([order, ends], 1).sort(1).values
        kept[r] = mine
        mine = mine.to(codes.device)
        full = budget // page * page
        new = weights[ids].transpose(0, 1).flatten(1).gather(1, mine)
        values = [_gathered(state, plane, ids).gather(1, mine[..., None].expand(-1, -1, case["dim"])) for plane in range(2)]
        for lo, hi in ((0, full), (full, budget)):
            if lo == hi:
                continue
            size = min(page, hi - lo)
            at = target[lo // page:-(-hi // page)]
            for plane in range(2):
                x = values[plane][:, lo:hi].reshape(kv, at.numel(), size, -1).transpose(0, 1)
                scale = _exact_scale(x, kind)
                part = codes[plane, at]
                part[:, :, :size] = _exact_code(x / scale[..., None, None], kind)
                codes[plane, at] = part
                scales[plane, at] = scale
            part = weights[at]
            part[:, :, :size] = new[:, lo:hi].reshape(kv, at.numel(), size).transpose(0, 1)
            weights[at] = part
    left = torch.tensor([min(n, budget) for n in lengths], dtype=torch.int32)
    return [codes, scales, weights, kept.int(), left]
