"""Blocks that come with scales that are no powers of two: append and evict round to the codes of the definition, to the bit, where
fp32 products and reciprocals end on the wrong side of a tie."""

import numpy as np
import pytest
import torch

from residualquant_b200.block_cache import BlockCache
from tests.test_gpu_block_cache import E4M3, INT8, ints, oracle_of, same_cache

pytestmark = pytest.mark.gpu

CODES = {INT8: np.arange(1, 128.0),
         E4M3: torch.arange(1, 127, dtype=torch.uint8).view(E4M3).double().numpy()}   # the positive values


def midpoints(dtype):
    return (CODES[dtype][1:] + CODES[dtype][:-1]) / 2


def ties(dtype, scale, act):
    """Values of `act` that lie halfway between two codes times `scale`, and that times the fp32 reciprocal do not."""
    x = midpoints(dtype) * float(scale)
    exact = torch.from_numpy(x).to(act).double().numpy() == x
    small = x <= CODES[dtype][-1] * 2.0 ** np.floor(np.log2(scale))      # the block keeps its scale
    moved = (x.astype(np.float32) * (np.float32(1) / np.float32(scale))).astype(np.float64) != midpoints(dtype)
    return x[exact & small], x[exact & small & moved]


def near_ties(dtype, border):
    """(code, ratio below 1 in fp32) whose product is above a midpoint (`border`: the largest code), but rounds to it in fp32."""
    found = []
    for tie in ([CODES[dtype][-1]] if border else midpoints(dtype)):
        for code in CODES[dtype]:
            ratio = np.float32(tie / code)
            ratio = ratio if float(ratio) * code > tie else np.nextafter(ratio, np.float32(np.inf))
            if (border or 0.5 < ratio < 1) and float(ratio) * code > tie and float(ratio * np.float32(code)) == tie:
                found.append((code, float(ratio)))
    return found


def raw(values, dtype):
    return torch.as_tensor(values, dtype=torch.float64).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("act", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,page", [(128, 16), (96, 32), (64, 16)])
def test_append_to_a_block_whose_scale_is_no_power_of_two(dtype, act, dim, page):
    scales = [s for s in (3, 7, 11, 13, 19, 41, 47, 55) if len(ties(dtype, s, act)[1])]
    assert scales, "no value in this test is in doubt"
    cache = BlockCache.allocate(len(scales), 1, dim, page, dtype, weights=True)
    table = ints([[i] for i in range(len(scales))])
    first = torch.ones(3 * len(scales), 1, dim, dtype=act, device="cuda")
    starts = lambda n: ints([n * i for i in range(len(scales) + 1)])
    cache.append(first, -first, starts(3), ints([3] * len(scales)), table)
    rows = []
    for i, scale in enumerate(scales):
        cache.scales[:, i] = float(scale)
        every, doubtful = ties(dtype, scale, act)
        row = np.resize(np.concatenate([doubtful, every, [scale, 0.7 * scale]]), 4 * dim)
        rows.append(torch.from_numpy(row * np.resize([1, -1, -1, 1, 1], 4 * dim)).to(act).reshape(4, 1, dim))
    key = torch.cat(rows).cuda()
    oracle = oracle_of(cache)
    cache.append(key, -key, starts(4), ints([7] * len(scales)), table)
    oracle.append(key, -key, starts(4).tolist(), [7] * len(scales), table.tolist())
    assert torch.equal(cache.scales, oracle.scale.float().cuda()) and float(cache.scales[0, 0]) == scales[0]
    same_cache(cache, oracle)


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("dim,page", [(128, 32), (96, 16), (64, 16)])
def test_append_rounds_earlier_tokens_again_from_a_scale_of_any_value(dtype, dim, page):
    found = near_ties(dtype, False)[:200]
    assert len(found) > 10
    cache = BlockCache.allocate(len(found), 1, dim, page, dtype)
    for i, (code, ratio) in enumerate(found):
        cache.codes[:, i] = raw(np.resize([code, -code, CODES[dtype][-1], 1], (page, dim)), dtype)
        cache.scales[:, i] = ratio
    oracle = oracle_of(cache)
    key = torch.full((len(found), 1, dim), float(CODES[dtype][-1]), dtype=torch.float16, device="cuda")   # needs a scale of 1
    args = list(range(len(found) + 1)), [6] * len(found), [[i] for i in range(len(found))]
    cache.append(key, -key, *(ints(a) for a in args))
    oracle.append(key, -key, *args)
    assert torch.all(cache.scales == 1.0)
    same_cache(cache, oracle)


@pytest.mark.parametrize("border", [False, True])
@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("dim,page", [(128, 16), (96, 32), (64, 32)])
def test_evict_from_blocks_with_scales_of_any_value(dtype, dim, page, border):
    """`border`: the largest value is above the range by less than fp32 shows, so the next power of two is needed."""
    found = near_ties(dtype, border)[:100]
    assert len(found) > 3
    cache = BlockCache.allocate(2 * len(found), 1, dim, page, dtype, weights=True)
    for i, (code, ratio) in enumerate(found):
        largest = code if border else CODES[dtype][-1]
        cache.codes[:, 2 * i:2 * i + 2] = raw(np.resize([code, -code, largest, CODES[dtype][0]], (page, dim)), dtype)
        cache.scales[:, 2 * i:2 * i + 2] = ratio
    cache.weights.copy_(torch.rand(cache.weights.shape, generator=torch.Generator().manual_seed(1)))
    oracle = oracle_of(cache)
    lengths, table = [page + 5] * len(found), [[2 * i, 2 * i + 1] for i in range(len(found))]
    kept, _ = cache.evict(ints(lengths), ints(table), page - 3, recent=2)
    want, _ = oracle.evict(lengths, table, page - 3, 0, 2)
    assert torch.equal(kept.cpu(), want)
    same_cache(cache, oracle)
