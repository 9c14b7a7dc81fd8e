"""The 8-bit block-scaled cache on the GPU against a plain 64-bit statement: append and evict to the bit, attention within
half a step of its output type and the roundings of its fp16 softmax weights."""

import random

import pytest
import torch

from residualquant_b200.block_cache import BlockCache
from tests import block_oracle

pytestmark = pytest.mark.gpu

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
DEVICE = "cuda"


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


class Batch:
    """Metadata of a batch: `counts` rows and `lengths` tokens a request, blocks shuffled over a pool."""

    def __init__(self, counts, lengths, page, seed=0, extra_blocks=3, width=None):
        rng = random.Random(seed)
        pages = [max(1, -(-max(n, 1) // page)) for n in lengths]
        self.blocks = sum(pages) + extra_blocks
        pool = list(range(self.blocks))
        rng.shuffle(pool)
        width = width or max(pages) + 1
        self.table = [[pool.pop() if i < n else -1 for i in range(width)] for n in pages]
        self.counts, self.lengths = list(counts), list(lengths)
        self.starts = [sum(counts[:i]) for i in range(len(counts) + 1)]
        self.meta = (ints(self.starts), ints(self.lengths), ints(self.table))


def make_cache(batch, heads, page, dim, dtype, weights=False, seed=0, garbage=True):
    """A cache whose every slot holds something: finite codes and power-of-two scales."""
    g = torch.Generator().manual_seed(seed)
    shape = (2, batch.blocks, heads, page, dim)
    if dtype == INT8:
        codes = torch.randint(-127, 128, shape, generator=g, dtype=torch.int8)
    else:
        codes = (torch.randn(shape, generator=g) * 90).clamp(-448, 448).to(E4M3)
    scales = 2.0 ** torch.randint(-8, -4, shape[:3], generator=g).float()
    w = torch.rand(shape[1:4], generator=g) ** 4 if weights else None
    if w is not None:
        w[torch.rand(w.shape, generator=g) < 0.2] = 0.0
    return BlockCache(codes.view(torch.uint8).cuda().view(dtype), scales.cuda(), w.cuda() if w is not None else None)


def oracle_of(cache):
    torch.cuda.synchronize()
    return block_oracle.Cache(cache.codes, cache.scales, cache.weights)


def same_cache(cache, oracle):
    torch.cuda.synchronize()
    assert torch.equal(cache.codes.view(torch.uint8).cpu(), oracle.byte)
    assert torch.equal(cache.scales.cpu().double(), oracle.scale)


def rows_like(count, heads, dim, act, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(count, heads, dim, generator=g) * scale).to(act).cuda()


def check_attention(cache, batch, query, *, scale=None, accumulate=False, pad=0, **more):
    """Runs the kernel and the oracle; returns the output."""
    scale = scale or cache.head_dim ** -0.5
    oracle = oracle_of(cache)
    out = torch.full_like(query, 77.0)
    lse = torch.full(query.shape[:2], 55.0, device=DEVICE)
    cache.attention(query, out, *batch.meta, softmax_scale=scale, lse=lse, accumulate=accumulate, **more)
    cache.attention_status()
    want, want_lse, magnitude, spread, added = oracle.attention(query, batch.starts, batch.lengths, batch.table, scale, accumulate,
                                                                more.get("max_seq_len"))
    real = batch.starts[-1]
    assert torch.all(out[real:] == 77.0) and torch.all(lse[real:] == 55.0), "padding rows were written"
    values = (oracle.value[1] * oracle.scale[1][..., None, None]).abs().max()
    limit = block_oracle.tolerance(want, magnitude, spread, max(batch.lengths), query.dtype, float(values))
    got = out.cpu().double()
    off = (got - want).abs()[:real]
    assert torch.all(off <= limit[:real]), f"off by {float((off / limit[:real]).max()):.3g} times the tolerance"
    got_lse = lse.cpu().double()[:real]
    assert torch.equal(torch.isinf(got_lse), torch.isinf(want_lse[:real]))
    fine = torch.isfinite(got_lse)
    slack = 2 * (cache.head_dim + 8) * 2.0 ** -24 * spread[:real] + 2.0 ** -18 + 2.0 ** -22 * want_lse[:real].abs()
    assert torch.all((got_lse - want_lse[:real]).abs()[fine] <= slack[fine])
    if accumulate:
        new = cache.weights.cpu().double()
        score = float(2 * (cache.head_dim + 8) * 2.0 ** -24 * spread.max() + 2.0 ** -17)
        assert torch.all((new - oracle.weight - added).abs() <= score * added + 2.0 ** -23 * (oracle.weight + added))
        assert torch.equal(new[added == 0], oracle.weight[added == 0]), "weights of unseen tokens changed"
    return out


# ---- append --------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dim,page,dtype,act,heads", [
    (128, 16, E4M3, torch.bfloat16, 2), (128, 32, INT8, torch.float16, 3), (96, 16, INT8, torch.bfloat16, 5),
    (96, 32, E4M3, torch.float16, 1), (64, 16, E4M3, torch.float16, 2), (64, 32, INT8, torch.bfloat16, 7),
])
def test_append_writes_the_codes_and_scales_of_the_definition(dim, page, dtype, act, heads):
    counts = [1, 0, 37, 16, 2, page, 1, 5]
    lengths = [1, 9, 37, 49, 18, 3 * page, page, 3]     # the last: five rows for three tokens
    batch = Batch(counts, lengths, page)
    cache = make_cache(batch, heads, page, dim, dtype, weights=True)
    oracle = oracle_of(cache)
    rows = batch.starts[-1] + 3                          # three padding rows
    key, value = rows_like(rows, heads, dim, act, 1, 3.0), rows_like(rows, heads, dim, act, 2)
    cache.append(key, value, *batch.meta)
    oracle.append(key, value, batch.starts, batch.lengths, batch.table)
    same_cache(cache, oracle)
    assert torch.equal(cache.weights.cpu().double(), oracle.weight)


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("page", [16, 32])
def test_append_token_by_token_rounds_earlier_tokens_again_when_a_scale_grows(dtype, page):
    batch = Batch([1, 1], [0, 0], page, width=3)
    batch.table = [[4, 2, 0], [1, 3, -1]]
    cache = make_cache(batch, 2, page, 64, dtype)
    cache = BlockCache(cache.codes[:, :5].contiguous(), cache.scales[:, :5].contiguous())
    oracle = oracle_of(cache)
    grown = 0
    for step in range(page + 5):
        key = rows_like(2, 2, 64, torch.bfloat16, 10 + step, 2.0 ** (step % 7 - 3))
        value = rows_like(2, 2, 64, torch.bfloat16, 99 + step, 0.0 if step < 3 else 1.0)
        before = cache.scales.clone()
        cache.append(key, value, ints([0, 1, 2]), ints([step + 1, step + 1]), ints(batch.table))
        oracle.append(key, value, [0, 1, 2], [step + 1, step + 1], batch.table)
        same_cache(cache, oracle)
        grown += int((cache.scales > before).sum())
    assert grown > 4


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("act", [torch.bfloat16, torch.float16])
def test_append_of_extreme_values(dtype, act):
    top = block_oracle.TOP[dtype]
    batch = Batch([16, 16, 16, 16, 16], [16] * 5, 16)
    cache = make_cache(batch, 1, 16, 64, dtype)
    oracle = oracle_of(cache)
    x = rows_like(80, 1, 64, act, 3)
    x[0:16] = 0.0                                        # a block of zeros
    x[16, 0, 0], x[17, 0, 1], x[18, 0, 2] = float("nan"), float("inf"), float("-inf")
    x[32:48] *= 2.0 ** -14                               # subnormal halves
    x[48:64] = torch.finfo(act).max
    x[64:80] = 0.0
    x[64, 0, 0], x[65, 0, 0] = top, torch.finfo(act).tiny  # exactly at the border, and the smallest normal
    cache.append(x, -x, *batch.meta)
    oracle.append(x, -x, batch.starts, batch.lengths, batch.table)
    same_cache(cache, oracle)
    assert torch.isfinite(cache.codes.float()).all()


def test_append_of_unaligned_and_strided_rows():
    batch = Batch([33, 1], [33, 40], 16)
    cache, other = (make_cache(batch, 3, 16, 96, E4M3) for _ in range(2))
    packed = rows_like(34, 7, 96, torch.bfloat16, 5)     # K and V are heads 1..3 and 4..6 of one packed tensor
    key, value = packed[:, 1:4], packed[:, 4:7]
    flat = torch.zeros(34 * 289 + 1, dtype=torch.bfloat16, device=DEVICE)[1:].view(34, 289)  # rows at odd addresses
    flat[:, :288] = key.reshape(34, 288)
    cache.append(key, value, *batch.meta)
    other.append(flat[:, :288].unflatten(1, (3, 96)), value, *batch.meta)
    oracle = oracle_of(make_cache(batch, 3, 16, 96, E4M3))
    oracle.append(key, value, batch.starts, batch.lengths, batch.table)
    same_cache(cache, oracle)
    same_cache(other, oracle)


def test_append_of_a_long_prompt_and_many_single_tokens():
    counts = [1] * 301 + [1531] + [0, 0, 2]
    lengths = [1 + 7 * i % 50 for i in range(301)] + [1600] + [0, 5, 2]
    batch = Batch(counts, lengths, 16, seed=4)
    cache = make_cache(batch, 1, 16, 64, INT8)
    oracle = oracle_of(cache)
    key, value = (rows_like(batch.starts[-1], 1, 64, torch.bfloat16, s, 2.0) for s in (1, 2))
    cache.append(key, value, *batch.meta)
    oracle.append(key, value, batch.starts, batch.lengths, batch.table)
    same_cache(cache, oracle)


def test_append_skips_blocks_outside_the_cache():
    batch = Batch([20, 20], [20, 20], 16)
    batch.table[0][0], batch.table[1][1] = batch.blocks, -7
    batch.meta = (batch.meta[0], batch.meta[1], ints(batch.table))
    cache = make_cache(batch, 1, 16, 64, E4M3)
    oracle = oracle_of(cache)
    key = rows_like(40, 1, 64, torch.float16, 1)
    cache.append(key, key, *batch.meta)
    oracle.append(key, key, batch.starts, batch.lengths, batch.table)
    same_cache(cache, oracle)
    cache.append(key, key, batch.meta[0], ints([20, 2000]), batch.meta[2])   # positions behind the table
    oracle.append(key[:20], key[:20], [0, 20], [20], batch.table[:1])
    same_cache(cache, oracle)


# ---- attention -----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("page,dtype,act", [(16, E4M3, torch.bfloat16), (32, E4M3, torch.float16), (16, INT8, torch.float16),
                                            (32, INT8, torch.bfloat16)])
@pytest.mark.parametrize("group,kv_heads", [(1, 3), (4, 2), (5, 1), (12, 1), (20, 1)])
def test_attention_of_single_tokens(dim, page, dtype, act, group, kv_heads):
    batch = Batch([1] * 9, [1, 0, 15, 16, 17, 63, 64, 65, 333], page, seed=dim)
    cache = make_cache(batch, kv_heads, page, dim, dtype)
    query = rows_like(9 + 2, kv_heads * group, dim, act, 7, 0.2)
    check_attention(cache, batch, query)


@pytest.mark.parametrize("dim,page,dtype,act", [(128, 16, E4M3, torch.bfloat16), (96, 32, INT8, torch.float16), (64, 32, E4M3, torch.bfloat16)])
@pytest.mark.parametrize("group", [1, 3, 8])
@pytest.mark.parametrize("most", [3, 9, 40])
def test_attention_of_several_rows_is_causal(dim, page, dtype, act, group, most):
    counts = [most, 1, 0, most // 2, most]
    lengths = [most, 70, 40, 200, max(2, most - 3)]      # the last: rows before the sequence's first token see nothing
    batch = Batch(counts, lengths, page, seed=most)
    cache = make_cache(batch, 2, page, dim, dtype)
    query = rows_like(batch.starts[-1] + 1, 2 * group, dim, act, 8, 0.2)
    check_attention(cache, batch, query)


@pytest.mark.parametrize("dim,page,dtype,group,counts", [(128, 16, E4M3, 4, [1, 1, 1, 1]), (128, 32, INT8, 1, [1, 1, 1, 1]), (96, 16, INT8, 2, [3, 1, 0, 5]),
                                                          (64, 32, E4M3, 12, [2, 1, 4, 33])])
def test_attention_accumulates_the_weights(dim, page, dtype, group, counts):
    batch = Batch(counts, [130, 1, 64, 500], page, seed=3)
    cache = make_cache(batch, 2, page, dim, dtype, weights=True)
    query = rows_like(batch.starts[-1] + 2, 2 * group, dim, torch.bfloat16, 9, 0.3)
    check_attention(cache, batch, query, accumulate=True)
    check_attention(cache, batch, query, accumulate=True, max_seq_len=500)


def test_attention_with_a_length_bound_below_a_length_sees_nothing_behind_it():
    batch = Batch([1, 2], [130, 90], 16)
    cache = make_cache(batch, 1, 16, 64, E4M3, weights=True)
    query = rows_like(3, 2, 64, torch.bfloat16, 9, 0.3)
    for accumulate in (False, True):
        check_attention(cache, batch, query, accumulate=accumulate, max_seq_len=100)


@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_attention_ignores_what_stands_behind_a_sequence(dtype):
    batch = Batch([1, 2], [21, 37], 16)
    cache = make_cache(batch, 2, 16, 128, dtype)
    query = rows_like(3, 2, 128, torch.bfloat16, 4, 0.2)
    first = check_attention(cache, batch, query)
    raw = cache.codes.view(torch.uint8)
    for r, n in enumerate(batch.lengths):
        raw[:, batch.table[r][n // 16], :, n % 16:] = 0x7F      # NaN in e4m3
    for b in set(range(batch.blocks)) - {x for row in batch.table for x in row}:
        raw[:, b] = 0xFF
        cache.scales[:, b] = float("nan")
    out = torch.full_like(query, 77.0)
    cache.attention(query, out, *batch.meta)
    assert torch.equal(out, first)


def test_attention_over_blocks_of_very_different_scales():
    """The large values stand where the softmax weight is nearly nothing, and the other way round."""
    batch = Batch([1, 1], [64, 640], 16)
    for k_step, v_step in ((0, 40), (0, -40), (1, 60), (-2, 30)):
        cache = make_cache(batch, 1, 16, 64, E4M3)
        query = rows_like(2, 2, 64, torch.bfloat16, 4, 0.5)
        for r in range(2):
            for i, b in enumerate(x for x in batch.table[r] if x >= 0):
                cache.scales[0, b] = 2.0 ** (-7 + k_step * (i % 3))
                cache.scales[1, b] = 2.0 ** (-7 + (v_step if i % 2 else 0))
        check_attention(cache, batch, query)


def test_attention_with_arbitrary_scales_and_large_or_small_queries():
    batch = Batch([1, 1, 1], [33, 100, 7], 32)
    cache = make_cache(batch, 2, 32, 96, INT8)
    cache.scales.mul_(torch.rand_like(cache.scales) + 0.5)
    for act, size in ((torch.bfloat16, 1e-30), (torch.bfloat16, 1e6), (torch.float16, 1e-4), (torch.float16, 1e4)):
        query = rows_like(3, 4, 96, act, 4, size)
        check_attention(cache, batch, query, scale=0.1 / size)
    query = rows_like(3, 4, 96, torch.bfloat16, 4)
    query[0] *= 0.0
    query[1, 0] *= 2.0 ** 60
    check_attention(cache, batch, query, scale=2.0 ** -58)


def test_attention_where_one_token_has_all_the_weight():
    batch = Batch([1], [700], 16)
    cache = make_cache(batch, 1, 16, 64, INT8)
    query = rows_like(1, 2, 64, torch.bfloat16, 4, 40.0)
    check_attention(cache, batch, query)


def test_attention_over_a_block_of_zeros_and_blocks_outside_the_cache():
    batch = Batch([1, 1], [80, 90], 16)
    cache = make_cache(batch, 1, 16, 128, E4M3)
    cache.codes.view(torch.uint8)[:, batch.table[0][2]] = 0
    cache.scales[:, batch.table[0][2]] = 1.0
    batch.table[0][3], batch.table[1][0] = -1, batch.blocks + 5
    batch.meta = (batch.meta[0], batch.meta[1], ints(batch.table))
    check_attention(cache, batch, rows_like(2, 1, 128, torch.bfloat16, 2, 0.3))


def test_attention_of_strided_rows():
    batch = Batch([1, 4], [50, 20], 16)
    cache = make_cache(batch, 2, 16, 128, E4M3)
    packed = rows_like(5, 8, 128, torch.bfloat16, 6, 0.2)
    plain = check_attention(cache, batch, packed[:, 2:6].contiguous())
    out = torch.zeros(5, 9, 128, dtype=torch.bfloat16, device=DEVICE)
    cache.attention(packed[:, 2:6], out[:, 3:7], *batch.meta)
    assert torch.equal(out[:, 3:7], plain) and torch.all(out[:, :3] == 0) and torch.all(out[:, 7:] == 0)
    table = torch.cat([batch.meta[2], batch.meta[2] * 0 - 1], 1)[:, :batch.meta[2].size(1)]  # a wider table's first columns
    again = torch.zeros_like(plain)
    cache.attention(packed[:, 2:6], again, batch.meta[0], batch.meta[1], table)
    assert torch.equal(again, plain)


def test_attention_writes_over_its_queries():
    batch = Batch([1, 3, 1], [700, 90, 2500], 16)
    cache = make_cache(batch, 2, 16, 128, INT8)
    query = rows_like(5, 8, 128, torch.bfloat16, 6, 0.2)
    want = torch.zeros_like(query)
    cache.attention(query, want, *batch.meta)
    cache.attention(query, query, *batch.meta)
    assert torch.equal(query, want)


def test_attention_of_many_requests():
    rng = random.Random(1)
    lengths = [rng.choice([0, 1, 5, 16, 30, 64, 100]) for _ in range(700)]
    counts = [rng.choice([0, 1, 1, 1, 2]) for _ in lengths]
    batch = Batch(counts, lengths, 16, seed=2)
    cache = make_cache(batch, 1, 16, 64, E4M3, weights=True)
    query = rows_like(batch.starts[-1] + 1, 2, 64, torch.bfloat16, 6, 0.2)
    check_attention(cache, batch, query, accumulate=True)


@pytest.mark.parametrize("requests,length,kv_heads,group,rows,dim,page,dtype,act", [
    (1, 40001, 1, 8, 1, 128, 16, E4M3, torch.bfloat16),      # one sequence is cut into hundreds of pieces
    (1, 20011, 3, 1, 1, 96, 32, INT8, torch.float16),
    (5, 9001, 2, 4, 1, 64, 16, E4M3, torch.bfloat16),
    (3, 7000, 2, 3, 7, 128, 16, INT8, torch.bfloat16),       # rows in two tiles of sixteen queries
    (40, 800, 2, 2, 1, 128, 32, E4M3, torch.float16),
])
def test_attention_over_long_sequences(requests, length, kv_heads, group, rows, dim, page, dtype, act):
    """Against float64 on the GPU, a head at a time."""
    lengths = [max(rows, length - 97 * i) for i in range(requests)]
    batch = Batch([rows] * requests, lengths, page, seed=length)
    cache = make_cache(batch, kv_heads, page, dim, dtype, weights=True)
    query = rows_like(rows * requests, kv_heads * group, dim, act, 3, 0.3)
    out, lse, start = torch.zeros_like(query), torch.zeros(query.shape[:2], device=DEVICE), cache.weights.double()
    for accumulate in (False, True):
        cache.attention(query, out, *batch.meta, lse=lse, accumulate=accumulate)
        cache.attention_status()
        added = torch.zeros_like(start)
        for r, n in enumerate(lengths):
            ids = torch.tensor([b for b in batch.table[r] if b >= 0], device=DEVICE)
            for h in range(kv_heads):
                keys, values = ((cache.codes.view(torch.uint8)[plane, ids, h].view(dtype).double() * cache.scales[plane, ids, h].double()[:, None, None])
                                .flatten(0, 1)[:n] for plane in range(2))
                q = query[rows * r:rows * (r + 1), h * group:(h + 1) * group].double()
                scores = torch.einsum("igd,td->igt", q, keys) * dim ** -0.5
                hidden = torch.arange(n, device=DEVICE) > (n - rows + torch.arange(rows, device=DEVICE))[:, None]
                scores = scores.masked_fill(hidden[:, None], float("-inf"))
                w = torch.softmax(scores, 2)
                want, magnitude = w @ values, w @ values.abs()
                spread = (q.abs() @ keys.abs().T).amax(2) * dim ** -0.5
                limit = block_oracle.tolerance(want, magnitude, spread, n, act, float(values.abs().max()))
                got = out[rows * r:rows * (r + 1), h * group:(h + 1) * group].double()
                assert torch.all((got - want).abs() <= limit)
                got = lse[rows * r:rows * (r + 1), h * group:(h + 1) * group].double()
                slack = 2 * (dim + 8) * 2.0 ** -24 * spread + 2.0 ** -18 + 2.0 ** -22 * got.abs()
                assert torch.all((got - torch.logsumexp(scores, 2)).abs() <= slack)
                sums = torch.zeros(ids.numel() * page, dtype=torch.float64, device=DEVICE)
                sums[:n] = w.sum((0, 1))
                added[ids, h] = sums.reshape(-1, page)
        if accumulate:
            score = 2 * (dim + 8) * 2.0 ** -24 * 40.0 + 2.0 ** -17      # scores here add up to less than 40 in magnitude
            assert float(spread.max()) < 40.0
            assert torch.all((cache.weights.double() - start - added).abs() <= score * added + 2.0 ** -22 * (start + added))


def test_attention_adds_up_the_weights_of_requests_that_share_blocks():
    batch = Batch([1, 1], [48, 48], 16)
    batch.table[1] = batch.table[0]
    batch.meta = (batch.meta[0], batch.meta[1], ints(batch.table))
    cache = make_cache(batch, 2, 16, 64, E4M3, weights=True)
    cache.weights.zero_()
    check_attention(cache, batch, rows_like(2, 4, 64, torch.bfloat16, 1, 0.3), accumulate=True)
    assert abs(float(cache.weights.sum()) - 2 * 4) < 1e-4


def test_attention_over_a_cache_beyond_32_bit_offsets():
    blocks, heads, dim = 70001, 16, 128                  # 4.6 GB of codes
    if torch.cuda.mem_get_info()[0] < 8 << 30:
        pytest.skip("not enough memory")
    codes = torch.zeros(2, blocks, heads, 16, dim, dtype=torch.int8, device=DEVICE)
    cache = BlockCache(codes, torch.ones(2, blocks, heads, device=DEVICE), torch.zeros(blocks, heads, 16, device=DEVICE))
    table = ints([[blocks - 1, blocks - 2, 5]])
    rows = rows_like(40, heads, dim, torch.bfloat16, 3)
    cache.append(rows, rows, ints([0, 40]), ints([40]), table)
    ids = table[0].long()
    small = BlockCache(codes[:, ids].contiguous(), cache.scales[:, ids].contiguous(), cache.weights[ids].contiguous())
    query = rows_like(1, heads, dim, torch.bfloat16, 4)
    outs = []
    for c, t in ((cache, table), (small, ints([[0, 1, 2]]))):
        out = torch.zeros_like(query)
        c.attention(query, out, ints([0, 1]), ints([40]), t, accumulate=True)
        kept, _ = c.evict(ints([40]), t, 20, recent=4)
        outs.append((out, kept))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    assert torch.equal(codes[:, ids], small.codes) and torch.equal(cache.weights[ids], small.weights)
    assert int(codes[:, :5].count_nonzero()) == 0
    values = small.codes[0, :2].float() * small.scales[0, :2, :, None, None]
    assert float(values.abs().max()) > 1.0


# ---- evict ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dim,page,dtype,heads", [(128, 16, E4M3, 2), (96, 32, INT8, 3), (64, 16, INT8, 1), (64, 32, E4M3, 2)])
@pytest.mark.parametrize("budget,sinks,recent", [(40, 4, 8), (33, 0, 0), (32, 16, 16), (1, 0, 1), (1, 0, 0), (100, 100, 0), (77, 0, 77)])
def test_evict_keeps_and_moves_the_tokens_of_the_definition(dim, page, dtype, heads, budget, sinks, recent):
    lengths = [200, 0, budget, budget + 1, 1, 131]
    batch = Batch([1] * 6, lengths, page, seed=budget)
    cache = make_cache(batch, heads, page, dim, dtype, weights=True, seed=budget)
    oracle = oracle_of(cache)
    kept, left = cache.evict(batch.meta[1], batch.meta[2], budget, sinks=sinks, recent=recent)
    want, want_left = oracle.evict(lengths, batch.table, budget, sinks, recent)
    assert torch.equal(kept.cpu(), want) and torch.equal(left.cpu(), want_left)
    same_cache(cache, oracle)
    assert torch.equal(cache.weights.cpu().double(), oracle.weight)


@pytest.mark.parametrize("kind", ["equal", "zero", "two values", "nan", "negative", "infinite", "ascending", "descending"])
def test_evict_of_special_weights(kind):
    batch = Batch([1, 1], [150, 140], 16)
    cache = make_cache(batch, 2, 16, 64, E4M3, weights=True)
    w = cache.weights
    if kind == "equal":
        w.fill_(0.37)
    elif kind == "zero":
        w.copy_(torch.where(w > 0.3, torch.zeros_like(w), -torch.zeros_like(w)))   # 0 and -0 are equal
    elif kind == "two values":
        w.copy_((w > 0.2).float() + 1.0)
    elif kind == "nan":
        w[w > 0.1] = float("nan")
    elif kind == "negative":
        w.sub_(0.3)
    elif kind == "infinite":
        w[w > 0.3] = float("inf")
        w[w == 0] = float("-inf")
    else:
        for r in range(2):
            order = torch.arange(160.0, device=DEVICE).reshape(10, 1, 16).expand(10, 2, 16) + 1
            n = len([b for b in batch.table[r] if b >= 0])
            w[batch.meta[2][r, :n].long()] = (order if kind == "ascending" else 200 - order)[:n]
    oracle = oracle_of(cache)
    kept, left = cache.evict(batch.meta[1], batch.meta[2], 50, sinks=3, recent=7)
    want, _ = oracle.evict(batch.lengths, batch.table, 50, 3, 7)
    assert torch.equal(kept.cpu(), want)
    same_cache(cache, oracle)


@pytest.mark.parametrize("requests,length,budget", [(1, 20011, 5003), (40, 700, 300), (300, 60, 33),
                                                    (1, 300007, 1000),      # more weights than eight CTAs hold
                                                    (76, 17003, 5000)])     # more than one holds
def test_evict_of_long_sequences_and_large_batches(requests, length, budget):
    batch = Batch([1] * requests, [length] * requests, 16, seed=1)
    cache = make_cache(batch, 2, 16, 64, INT8, weights=True)
    before = cache.codes.float() * cache.scales[..., None, None]
    weights = cache.weights.clone()
    kept, left = cache.evict(batch.meta[1], batch.meta[2], budget, sinks=4, recent=20)
    table = batch.meta[2].long()
    w = weights[table.clamp(min=0)].permute(0, 2, 1, 3).flatten(2)[..., :length].clone()
    w[..., :4] = w[..., -20:] = float("inf")
    want = torch.sort(w, dim=2, descending=True, stable=True).indices[..., :budget].sort(2).values
    assert torch.equal(kept.long(), want)
    after = cache.codes.float() * cache.scales[..., None, None]
    head = torch.arange(2, device=DEVICE)[None, :, None]

    def tokens(values, index):   # values of the tokens at positions `index` [requests, heads, n]
        return values[:, torch.gather(table[:, None].expand(-1, 2, -1), 2, index // 16), head, index % 16]

    moved, source = tokens(after, torch.arange(budget, device=DEVICE).expand_as(want)), tokens(before, want)
    # a code is rounded to its block's new scale, which is at most the largest source scale of the block
    assert float((moved - source).abs().max()) <= 0.5 * float(cache.scales.max())
    assert torch.equal(cache.weights[torch.gather(table[:, None].expand(-1, 2, -1), 2, torch.arange(budget, device=DEVICE).expand_as(want) // 16),
                                     head, torch.arange(budget, device=DEVICE).expand_as(want) % 16],
                       weights[torch.gather(table[:, None].expand(-1, 2, -1), 2, want // 16), head, want % 16])


# ---- together ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_a_decode_run_with_eviction(dtype):
    """Prompts, then steps of append and attention that accumulate, an eviction in between, and steps after it."""
    page, heads, group, dim, budget = 16, 2, 3, 64, 48
    lengths, table = [30, 70, 5], [[i * 6 + j for j in range(6)] for i in range(3)]
    cache = BlockCache.allocate(18, heads, dim, page, dtype, weights=True)
    mirror = oracle_of(cache)
    starts = [0, 30, 100, 105]
    for step in range(8):
        if step:
            starts, lengths = [0, 1, 2, 3], [n + 1 for n in lengths]
        key, value = (rows_like(starts[-1], heads, dim, torch.bfloat16, 50 * step + s) for s in (1, 2))
        query = rows_like(starts[-1], heads * group, dim, torch.bfloat16, 50 * step + 3)
        meta = ints(starts), ints(lengths), ints(table)
        cache.append(key, value, *meta)
        mirror.append(key, value, starts, lengths, table)
        same_cache(cache, mirror)
        batch = Batch([0], [0], page)
        batch.starts, batch.lengths, batch.table, batch.meta, batch.blocks = starts, lengths, table, meta, 18
        check_attention(cache, batch, query, accumulate=True)
        mirror.weight = cache.weights.cpu().double()
        if step in (2, 5):
            kept, left = cache.evict(meta[1], meta[2], budget, sinks=2, recent=9)
            want, want_left = mirror.evict(lengths, table, budget, 2, 9)
            assert torch.equal(kept.cpu(), want)
            same_cache(cache, mirror)
            lengths = left.tolist()


def test_calls_are_captured_and_replayed_with_new_lengths():
    batch = Batch([1, 1, 1], [40, 70, 3], 16, width=8)
    batch.table = [[3 * j + i for j in range(8)] for i in range(3)]
    cache = BlockCache.allocate(24, 2, 128, 16, E4M3, weights=True)
    fill = rows_like(113, 2, 128, torch.bfloat16, 1)
    cache.append(fill, fill.flip(0), ints([0, 40, 110, 113]), ints([40, 70, 3]), ints(batch.table))
    starts, lengths, table = ints([0, 1, 2, 3]), ints([41, 71, 4]), ints(batch.table)
    key, value, query = (rows_like(3, h, 128, torch.bfloat16, 5) for h in (2, 2, 4))
    out, lse = torch.zeros_like(query), torch.zeros(3, 4, device=DEVICE)
    kept, left = torch.zeros(3, 2, 32, dtype=torch.int32, device=DEVICE), ints([0, 0, 0])
    torch.cuda.synchronize()
    saved = [t.clone() for t in (cache.codes, cache.scales, cache.weights)]

    def step():
        cache.append(key, value, starts, lengths, table)
        cache.attention(query, out, starts, lengths, table, lse=lse, accumulate=True)
        cache.evict(lengths, table, 32, recent=4, kept=kept, new_lens=left)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for lens in ([41, 71, 4], [100, 2, 31], [1, 128, 33]):
        lengths.copy_(ints(lens))
        results = []
        for go in (step, graph.replay):
            for t, s in zip((cache.codes, cache.scales, cache.weights), saved):
                t.view(torch.uint8).copy_(s.view(torch.uint8))
            for t in (out, lse, kept, left):
                t.zero_()
            go()
            torch.cuda.synchronize()
            results.append([t.clone() for t in (cache.codes.view(torch.uint8), cache.scales, cache.weights, out, lse, kept, left)])
        assert all(torch.equal(a, b) for a, b in zip(*results))


def test_two_captured_graphs_are_replayed_at_once():
    """Each graph has scratch memory of its own: replayed on two streams they give what they give alone."""
    batch = Batch([1] * 6, [1500] * 6, 16)
    cache = make_cache(batch, 2, 16, 128, INT8)
    queries, outs, wants, graphs = [], [], [], []
    for s in (1, 2):
        queries.append(rows_like(6, 8, 128, torch.bfloat16, s, 0.2))
        outs.append(torch.zeros_like(queries[-1]))
        wants.append(torch.zeros_like(queries[-1]))
        cache.attention(queries[-1], wants[-1], *batch.meta)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            for _ in range(4):
                outs[-1].zero_()
                cache.attention(queries[-1], outs[-1], *batch.meta)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, wants))


def test_two_streams_share_nothing():
    """Calls on two streams at once, each on its own rows of the same cache, give what they give one after the other."""
    batch = Batch([1] * 8, [900] * 8, 16)
    cache = make_cache(batch, 2, 16, 128, E4M3, weights=True)
    queries = [rows_like(8, 8, 128, torch.bfloat16, s, 0.2) for s in (1, 2)]
    wants, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for q in queries:
        wants.append(torch.zeros_like(q))
        cache.attention(q, wants[-1], *batch.meta)
    outs = [[torch.zeros_like(q) for _ in range(20)] for q in queries]
    torch.cuda.synchronize()
    for i in range(20):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                cache.attention(queries[s], outs[s][i], *batch.meta)
    torch.cuda.synchronize()
    assert all(torch.equal(o, wants[s]) for s in range(2) for o in outs[s])


def test_repeated_calls_give_the_same_bits():
    batch = Batch([1, 2, 5], [3000, 77, 900], 16)
    cache = make_cache(batch, 2, 16, 128, INT8, weights=True)
    query = rows_like(8, 8, 128, torch.bfloat16, 3, 0.2)
    start = cache.weights.clone()
    results = []
    for _ in range(5):
        cache.weights.copy_(start)
        out = torch.zeros_like(query)
        cache.attention(query, out, *batch.meta, accumulate=True)
        results.append((out, cache.weights.clone()))
    assert all(torch.equal(a, b) for r in results[1:] for a, b in zip(r, results[0]))


def test_empty_calls_do_nothing():
    cache = BlockCache.allocate(4, 2, 64, 16, INT8, weights=True)
    before = cache.codes.clone()
    none = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device=DEVICE)
    cache.append(none, none, ints([0, 0]), ints([5]), ints([[1]]))
    cache.attention(none, none, ints([0, 0]), ints([5]), ints([[1]]))
    kept, left = cache.evict(ints([]), ints([]).reshape(0, 1), 4)
    assert kept.shape == (0, 2, 4) and left.numel() == 0
    one = rows_like(1, 2, 64, torch.bfloat16, 1)
    out = torch.full_like(one, 3.0)
    cache.attention(one, out, ints([0, 0]), ints([5]), ints([[1]]))            # only a padding row
    cache.attention(one, out, ints([0, 0]), ints([5]), ints([[1]]).reshape(1, 1)[:, :0])
    assert torch.all(out == 3.0)
    cache.attention(one, out, ints([0, 1]), ints([5]), ints([[1]])[:, :0])     # a row whose table has no block
    assert torch.all(out == 0.0) and torch.equal(cache.codes, before)


def refusals(cache):
    one = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=cache.device)
    starts, lengths, table = (t.to(cache.device) for t in (torch.tensor([0, 1, 2]).int(), torch.tensor([4, 4]).int(), torch.tensor([[1], [2]]).int()))
    good = (starts, lengths, table)
    yield lambda: cache.append(one.float(), one, *good)
    yield lambda: cache.append(one, one[:1], *good)
    yield lambda: cache.append(one, one.half(), *good)
    yield lambda: cache.append(one[:, :1], one, *good)
    yield lambda: cache.append(one.transpose(0, 1), one, *good)
    yield lambda: cache.append(one.cpu() if cache.device.type == "cuda" else one.to("meta"), one, *good)
    yield lambda: cache.append(one, one, starts.long(), lengths, table)
    yield lambda: cache.append(one, one, starts[:2], lengths, table)
    yield lambda: cache.append(one, one, starts, lengths, table[:1])
    yield lambda: cache.append(one, one, starts, lengths, table.float())
    yield lambda: cache.append(one, one, starts, lengths[::2].repeat(2)[::2], table)
    yield lambda: cache.attention(torch.zeros(2, 3, 64, dtype=torch.bfloat16, device=cache.device), one, *good)
    yield lambda: cache.attention(one, one.half(), *good)
    yield lambda: cache.attention(one[0], one[0], *good)
    yield lambda: cache.attention(one, one, *good, lse=torch.zeros(2, 3, device=cache.device))
    yield lambda: cache.attention(one, one, *good, softmax_scale=0.0)
    yield lambda: cache.attention(one, one, *good, softmax_scale=float("nan"))
    yield lambda: cache.attention(one, one, *good, max_seq_len=0)
    yield lambda: cache.attention(torch.zeros(2 * 132 + 4, dtype=torch.bfloat16, device=cache.device)[4:].view(2, 132)[:, :128].unflatten(1, (2, 64)), one, *good)
    yield lambda: cache.evict(lengths, table, 0)
    yield lambda: cache.evict(lengths, table, 4, sinks=3, recent=2)
    yield lambda: cache.evict(lengths, table, 4, sinks=-1)
    yield lambda: cache.evict(lengths, table, 4, new_lens=lengths)
    yield lambda: cache.evict(lengths, table, 4, kept=torch.zeros(2, 2, 5, dtype=torch.int32, device=cache.device))
    bare = BlockCache(cache.codes, cache.scales)
    yield lambda: bare.evict(lengths, table, 4)
    yield lambda: bare.attention(one, one, *good, accumulate=True)
    yield lambda: BlockCache(cache.codes.view(torch.uint8), cache.scales)
    yield lambda: BlockCache(cache.codes[:, :, :, :8].contiguous(), cache.scales)
    yield lambda: BlockCache(cache.codes[..., :32].contiguous(), cache.scales)
    yield lambda: BlockCache(cache.codes.transpose(1, 2), cache.scales)
    yield lambda: BlockCache(cache.codes, cache.scales.double())
    yield lambda: BlockCache(cache.codes, cache.scales, cache.scales)


def test_rejected_arguments_raise():
    cache = BlockCache.allocate(4, 2, 64, 16, INT8, weights=True)
    for i, call in enumerate(refusals(cache)):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was accepted")
