"""Block-cache attention keeps its softmax weights to 22 bits: value sums that nearly cancel show what a weight is off by."""

import pytest
import torch

from tests.test_gpu_block_cache import E4M3, INT8, Batch, make_cache, oracle_of, rows_like

pytestmark = pytest.mark.gpu


def cancelling_limit(want, magnitude, spread, dim, dtype, tokens, top):
    """How far an output may be off.  Half a step of the output's type.  Each weight, relative to itself: a score off by at most
    dim + 8 roundings of 2^-24 of the terms' sum `spread`, twice; exponents of at most 2^5 in magnitude, rounded twice on the way
    in and twice on the way out, and two exponentials of 2 units each, together below 2^-17; two fp16 parts, 2^-22; at most
    tokens / 64 + 8 additions of 2^-22 in a warp and over the warps.  And 2^-31 of the largest value for each token, where the
    fp16 parts end (2^-25 each, of a largest weight of at least 2^7)."""
    relative = 2.0 ** -17 + (tokens / 64 + 9) * 2.0 ** -22 + (2 * (dim + 8) * 2.0 ** -24 * spread)[..., None]
    return torch.finfo(dtype).eps / 2 * want.abs() + relative * magnitude * (1 + 2.0 ** -8) + tokens * 2.0 ** -31 * top


@pytest.mark.parametrize("dim,page,dtype,group", [(128, 16, E4M3, 4), (128, 32, INT8, 12), (96, 16, INT8, 5), (96, 32, E4M3, 16), (64, 16, E4M3, 8),
                                                  (64, 32, INT8, 1)])
@pytest.mark.parametrize("act", [torch.float16, torch.bfloat16])
def test_value_sums_that_nearly_cancel(dim, page, dtype, group, act):
    batch = Batch([1] * 6, [2, 3, 9, 17, 40, 300], page, seed=dim + page)
    cache = make_cache(batch, 2, page, dim, dtype, seed=group)
    g = torch.Generator().manual_seed(5)
    signs = torch.where(torch.rand(cache.codes.shape[1:], generator=g) < 0.5, -1.0, 1.0).cuda()
    level = 100.0 + torch.randint(0, 2, cache.codes.shape[1:], generator=g).cuda() * 4.0    # codes of both types
    cache.codes[1] = (signs * level).to(dtype)
    cache.scales[1] = 2.0 ** -7
    query = rows_like(6, 2 * group, dim, act, 11, 0.2)
    out = torch.zeros_like(query)
    cache.attention(query, out, *batch.meta)
    want, _, magnitude, spread, _ = oracle_of(cache).attention(query, batch.starts, batch.lengths, batch.table, dim ** -0.5)
    top = 104.0 * 2.0 ** -7
    lengths = torch.tensor(batch.lengths, dtype=torch.float64)[:, None, None]
    limit = cancelling_limit(want, magnitude, spread, dim, act, lengths, top)
    assert float((magnitude / want.abs().clamp(min=1e-30)).max()) > 1000          # the sums do cancel
    off = (out.cpu().double() - want).abs()
    assert torch.all(off <= limit), f"off by {float((off / limit).max()):.3g} times the tolerance"
