"""The block cache at the sizes that choose other launch shapes: prompts of thousands of rows, evictions by clusters of CTAs in many
waves, attention pieces of thousands of tokens, block tables far wider than their sequences.  Against the definitions in 64 bits,
on the GPU: append and evict to the bit, attention within the tolerances of `block_oracle`."""

import random

import pytest
import torch

from residualquant_b200.block_cache import BlockCache
from tests import block_oracle
from tests.test_gpu_block_cache import DEVICE, E4M3, INT8, Batch, check_attention, ints, make_cache, oracle_of, rows_like

pytestmark = pytest.mark.gpu


def random_cache(blocks, heads, page, dim, dtype, weights=False, seed=0):
    """A cache whose every slot holds something: finite codes, power-of-two scales, heavy-tailed weights."""
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    shape = (2, blocks, heads, page, dim)
    if dtype == INT8:
        codes = torch.randint(-127, 128, shape, generator=g, dtype=torch.int8, device=DEVICE)
    else:
        codes = (torch.randn(shape, generator=g, device=DEVICE) * 90).clamp(-448, 448).to(E4M3)
    scales = 2.0 ** torch.randint(-9, -5, shape[:3], generator=g, device=DEVICE).float()
    w = torch.rand(shape[1:4], generator=g, device=DEVICE) ** 4 if weights else None
    return BlockCache(codes, scales, w)


def shuffled_table(pages, blocks, width, seed):
    pool = list(range(blocks))
    random.Random(seed).shuffle(pool)
    return [[pool.pop() if i < n else -1 for i in range(width)] for n in pages]


def needed(amax, dtype):
    """The smallest power of two (from 2^-100 on) with amax <= top * it; 1 for 0."""
    top, at = torch.frexp(torch.tensor(block_oracle.TOP[dtype], dtype=torch.float64))
    mantissa, exponent = torch.frexp(amax)
    exponent = (exponent - int(at) + (mantissa > float(top)).int()).clamp(min=-100)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), exponent), torch.ones_like(amax))


def copy_of(cache):
    return [cache.codes.view(torch.uint8).clone(), cache.scales.clone(), cache.weights.clone() if cache.weights is not None else None]


def same(cache, want):
    assert torch.equal(cache.scales, want[1])
    assert torch.equal(cache.codes.view(torch.uint8), want[0])
    assert want[2] is None or torch.equal(cache.weights, want[2])


def values_of(raw, scales, dtype, plane, block):
    return raw[plane, block].view(dtype).double() * scales[plane, block].double()[..., None, None]


def appended(cache, key, value, starts, lengths, table):
    """What a call leaves: bytes, scales, weights."""
    dtype, page = cache.codes.dtype, cache.block_size
    codes, scales, weights = copy_of(cache)
    for r, length in enumerate(lengths):
        first = length - (starts[r + 1] - starts[r])
        for b in range(max(0, first) // page, -(-length // page)):
            lo, hi = max(b * page, first), min((b + 1) * page, length)
            if b >= len(table[r]) or not 0 <= table[r][b] < cache.num_blocks or lo >= hi:
                continue
            block, old = table[r][b], max(0, lo - b * page)
            for plane, source in enumerate((key, value)):
                x = source[starts[r] + lo - first:starts[r] + hi - first].double().transpose(0, 1)   # [heads, tokens, channels]
                finite = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax((1, 2))
                scale, before = needed(finite, dtype), scales[plane, block].double()
                if old:
                    scale = torch.where(finite > 0, torch.maximum(scale, before), before)
                    held = codes[plane, block, :, :old].view(dtype).double() * (before / scale)[:, None, None]
                    again = block_oracle.raw(block_oracle.rounded(held, dtype), dtype)
                    codes[plane, block, :, :old] = torch.where((scale > before)[:, None, None], again, codes[plane, block, :, :old])
                codes[plane, block, :, old:old + hi - lo] = block_oracle.raw(block_oracle.rounded(x / scale[:, None, None], dtype), dtype)
                scales[plane, block] = scale.float()
            if weights is not None:
                weights[block, :, old:old + hi - lo] = 0.0
    return codes, scales, weights


@pytest.mark.parametrize("heads,dim,page,dtype,act,requests,rows", [
    (13, 64, 16, E4M3, torch.bfloat16, 24, 9200),      # a warp walks over 16 rows and takes four heads and planes, the last one two
    (13, 64, 32, INT8, torch.float16, 10, 9200),       # 32 rows
    (7, 96, 16, INT8, torch.bfloat16, 40, 1500),       # 4 rows, one head and plane
    (3, 128, 32, E4M3, torch.float16, 30, 2600),       # 4 rows
    (7, 64, 16, INT8, torch.bfloat16, 2100, 2100),     # one row, four heads and planes
    (16, 128, 16, E4M3, torch.bfloat16, 900, 4000),    # 4 rows over many requests
])
def test_append_of_prompts(heads, dim, page, dtype, act, requests, rows):
    rng = random.Random(heads * rows)
    cuts = sorted(rng.randrange(rows + 1) for _ in range(requests - 1))
    if requests == rows:
        cuts = list(range(1, rows))
    starts = [0] + cuts + [rows]                                                    # some requests have no rows
    counts = [b - a for a, b in zip(starts, starts[1:])]
    before = [rng.choice([0, 0, rng.randrange(1, 50)]) for _ in counts]             # many begin inside a block
    lengths = [n + b for n, b in zip(counts, before)]
    lengths[1] = max(0, counts[1] - 5)                                              # rows before the sequence's first token
    pages = [-(-max(n, 1) // page) for n in lengths]
    blocks = sum(pages) + 2
    table = shuffled_table(pages, blocks, max(pages), rows)
    table[2][0], table[3][0] = -1, blocks                                           # blocks outside the cache
    cache = random_cache(blocks, heads, page, dim, dtype, weights=True, seed=rows)
    g = torch.Generator(device=DEVICE).manual_seed(1)
    key, value = (torch.randn(rows + 3, heads, dim, generator=g, device=DEVICE) * 2.0 ** torch.randint(-6, 3, (rows + 3, heads, 1), generator=g, device=DEVICE)
                  for _ in range(2))
    key, value = key.to(act), value.to(act)
    value[7, 0, 1], value[40, 1, 2], key[41, 2, 3] = float("nan"), float("inf"), float("-inf")
    want = appended(cache, key, value, starts, lengths, table)
    cache.append(key, value, ints(starts), ints(lengths), ints(table))
    same(cache, want)


def evicted(cache, lengths, table, budget, sinks, recent):
    """What a call leaves (bytes, scales, weights), the kept positions and the new lengths."""
    dtype, page, heads, dim = cache.codes.dtype, cache.block_size, cache.kv_heads, cache.head_dim
    codes, scales, weights = copy_of(cache)
    kept = torch.full((len(lengths), heads, budget), -1, dtype=torch.int64, device=DEVICE)
    for r, n in enumerate(lengths):
        kept[r, :, :min(n, budget)] = torch.arange(min(n, budget), device=DEVICE)
        if n <= budget:
            continue
        ids = torch.tensor(table[r][:-(-n // page)], device=DEVICE)
        w = cache.weights[ids].transpose(0, 1).flatten(1)[:, :n]
        middle = w[:, sinks:n - recent]
        order = torch.argsort(middle, dim=1, descending=True, stable=True)[:, :budget - sinks - recent] + sinks
        ends = torch.cat([torch.arange(sinks, device=DEVICE), torch.arange(n - recent, n, device=DEVICE)]).expand(heads, -1)
        mine = torch.cat([order, ends], 1).sort(1).values
        kept[r] = mine
        moved = w.gather(1, mine)
        for plane in range(2):
            x = values_of(cache.codes.view(torch.uint8), cache.scales, dtype, plane, ids).transpose(0, 1).flatten(1, 2)
            x = x.gather(1, mine[..., None].expand(-1, -1, dim))
            for b in range(0, budget, page):
                part, block = x[:, b:b + page], int(ids[b // page])
                scale = needed(part.abs().amax((1, 2)), dtype)
                codes[plane, block, :, :part.shape[1]] = block_oracle.raw(block_oracle.rounded(part / scale[:, None, None], dtype), dtype)
                scales[plane, block] = scale.float()
        for b in range(0, budget, page):
            part = moved[:, b:b + page]
            weights[int(ids[b // page]), :, :part.shape[1]] = part
    return (codes, scales, weights), kept.int(), ints([min(n, budget) for n in lengths])


@pytest.mark.parametrize("requests,length,budget,heads", [
    (1, 9001, 4099, 2),        # eight CTAs for each head, several waves, the last block partly filled
    (1, 4500, 1000, 3),        # four
    (2, 2500, 777, 1),         # two
    (3, 900, 300, 2),          # one of sixteen warps
    (80, 700, 333, 2),         # one of eight warps
])
@pytest.mark.parametrize("dim,page,dtype", [(128, 16, E4M3), (128, 32, INT8), (96, 32, E4M3), (96, 16, INT8), (64, 16, E4M3), (64, 32, INT8)])
def test_evict_by_clusters_and_in_waves(requests, length, budget, heads, dim, page, dtype):
    lengths = [length - 13 * (i % 20) if i % 7 != 5 else budget for i in range(requests)]
    pages = [-(-n // page) for n in lengths]
    table = shuffled_table(pages, sum(pages) + 3, max(pages), length)
    cache = random_cache(sum(pages) + 3, heads, page, dim, dtype, weights=True, seed=dim + page)
    cache.weights[torch.rand(cache.weights.shape, device=DEVICE, generator=torch.Generator(device=DEVICE).manual_seed(2)) < 0.3] = 0.25    # ties
    want, kept, left = evicted(cache, lengths, table, budget, 4, 50)
    got = cache.evict(ints(lengths), ints(table), budget, sinks=4, recent=50)
    assert torch.equal(got[0], kept) and torch.equal(got[1], left)
    same(cache, want)


def test_evict_puts_nan_behind_everything():
    batch = Batch([1], [60], 16)
    cache = make_cache(batch, 1, 16, 64, E4M3, weights=True)
    at = [(batch.table[0][t // 16], 0, t % 16) for t in range(60)]
    for t, place in enumerate(at):
        cache.weights[place] = float("nan") if t % 3 == 0 else float("-inf")       # 20 of NaN, 40 of -inf
    kept, _ = cache.evict(batch.meta[1], batch.meta[2], 45)
    lower = [t for t in range(60) if t % 3] + [t for t in range(60) if t % 3 == 0][:5]
    assert kept[0, 0].tolist() == sorted(lower)


def attend(cache, query, starts, lengths, table, accumulate=False, **more):
    """Runs a call and holds its outputs and weights against float64, a request and head at a time."""
    dim, dtype, page, heads = cache.head_dim, cache.codes.dtype, cache.block_size, cache.kv_heads
    group = query.shape[1] // heads
    before = cache.weights.double() if accumulate else None
    out, lse = torch.full_like(query, 77.0), torch.full(query.shape[:2], 55.0, device=DEVICE)
    cache.attention(query, out, ints(starts), ints(lengths), ints(table), lse=lse, accumulate=accumulate, **more)
    cache.attention_status()
    real = starts[-1]
    assert torch.all(out[real:] == 77.0) and torch.all(lse[real:] == 55.0)
    added = torch.zeros_like(before) if accumulate else None
    most = 0.0
    for r, n in enumerate(lengths):
        rows = starts[r + 1] - starts[r]
        ids = torch.tensor(table[r][:-(-n // page)], device=DEVICE)
        for h in range(heads):
            keys, values = ((cache.codes.view(torch.uint8)[plane, ids, h].view(dtype).double() * cache.scales[plane, ids, h].double()[:, None, None])
                            .flatten(0, 1)[:n] for plane in range(2))
            mine = slice(starts[r], starts[r + 1]), slice(h * group, (h + 1) * group)
            q = query[mine].double()
            scores = torch.einsum("igd,td->igt", q, keys) * dim ** -0.5
            hidden = torch.arange(n, device=DEVICE) > (n - rows + torch.arange(rows, device=DEVICE))[:, None]
            scores = scores.masked_fill(hidden[:, None], float("-inf"))
            w = torch.softmax(scores, 2)
            want, magnitude = w @ values, w @ values.abs()
            spread = (q.abs() @ keys.abs().T).amax(2) * dim ** -0.5
            most = max(most, float(spread.max()))
            limit = block_oracle.tolerance(want, magnitude, spread, n, query.dtype, float(values.abs().max()))
            assert torch.all((out[mine].double() - want).abs() <= limit), (r, h)
            slack = 2 * (dim + 8) * 2.0 ** -24 * spread + 2.0 ** -18 + 2.0 ** -22 * lse[mine].double().abs()
            assert torch.all((lse[mine].double() - torch.logsumexp(scores, 2)).abs() <= slack), (r, h)
            if accumulate:
                sums = torch.zeros(ids.numel() * page, dtype=torch.float64, device=DEVICE)
                sums[:n] = w.sum((0, 1))
                added[ids, h] = sums.reshape(-1, page)
    if accumulate:
        # each weight by its score's error, and the sums' last bits: a token adds up at most rows x group weights
        score = 2 * (dim + 8) * 2.0 ** -24 * most + 2.0 ** -17
        assert torch.all((cache.weights.double() - before - added).abs() <= score * added + 2.0 ** -22 * (before + added))
    return out


@pytest.mark.parametrize("requests,longest,shortest,kv_heads,group,rows,dim,page,dtype,act", [
    (40, 6000, 2500, 16, 1, 1, 64, 16, E4M3, torch.bfloat16),     # pieces of more than 4096 tokens: a warp's pages come in three windows
    (40, 6100, 2500, 16, 12, 1, 64, 32, INT8, torch.float16),     # the same with sixteen queries
    (40, 5003, 4000, 16, 2, 2, 96, 16, INT8, torch.bfloat16),
    (70, 2300, 2100, 16, 6, 1, 128, 32, E4M3, torch.bfloat16),    # about two items for each CTA, five to eight queries
    (30, 1000, 600, 8, 3, 1, 128, 16, INT8, torch.bfloat16),      # 513 to 1024 tokens: an item for each CTA, none is cut
    (30, 1000, 600, 8, 10, 1, 64, 16, E4M3, torch.float16),
    (20, 1024, 513, 12, 1, 3, 96, 32, E4M3, torch.bfloat16),
    (9, 1000, 600, 2, 4, 1, 128, 16, INT8, torch.bfloat16),       # too few of them: cut
    (100, 1000, 600, 16, 1, 1, 64, 16, INT8, torch.bfloat16),     # too many: cut
])
def test_attention_over_long_pieces(requests, longest, shortest, kv_heads, group, rows, dim, page, dtype, act):
    rng = random.Random(longest + dim)
    lengths = [longest] + [rng.randint(shortest, longest) for _ in range(requests - 1)]
    pages = [-(-n // page) for n in lengths]
    table = shuffled_table(pages, sum(pages) + 3, max(pages), longest)
    cache = random_cache(sum(pages) + 3, kv_heads, page, dim, dtype, weights=True, seed=longest)
    query = rows_like(rows * requests + 2, kv_heads * group, dim, act, 3, 0.3)
    starts = [rows * i for i in range(requests + 1)]
    plain = attend(cache, query, starts, lengths, table)
    assert torch.equal(attend(cache, query, starts, lengths, table, accumulate=True), plain)


@pytest.mark.parametrize("width", [2049, 8192])
def test_tables_far_wider_than_their_sequences(width):
    """What an engine passes: one table as wide as its longest allowed sequence."""
    lengths, counts = [97, 1, 400, 30], [1, 1, 3, 0]
    batch = Batch(counts, lengths, 16, width=width)
    cache = make_cache(batch, 2, 16, 128, E4M3, weights=True)
    oracle = oracle_of(cache)
    rows = rows_like(5, 2, 128, torch.bfloat16, 1)
    cache.append(rows, -rows, *batch.meta)
    oracle.append(rows, -rows, batch.starts, lengths, batch.table)
    assert torch.equal(cache.codes.view(torch.uint8).cpu(), oracle.byte) and torch.equal(cache.scales.cpu().double(), oracle.scale)
    query = rows_like(6, 8, 128, torch.bfloat16, 2, 0.3)
    check_attention(cache, batch, query)
    check_attention(cache, batch, query, accumulate=True)
    check_attention(cache, batch, query, accumulate=True, max_seq_len=400)
    oracle = oracle_of(cache)
    kept, left = cache.evict(batch.meta[1], batch.meta[2], 61, sinks=2, recent=9)
    want, want_left = oracle.evict(lengths, batch.table, 61, 2, 9)
    assert torch.equal(kept.cpu(), want) and torch.equal(left.cpu(), want_left)
    assert torch.equal(cache.codes.view(torch.uint8).cpu(), oracle.byte) and torch.equal(cache.scales.cpu().double(), oracle.scale)
