"""Calls of the block cache that follow one another."""

import pytest
import torch

from tests.test_gpu_block_cache import E4M3, Batch, check_attention, make_cache, rows_like

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("refused", ["scale", "expanded rows"])
def test_a_refused_attention_call_leaves_later_ones_alone(refused):
    batch = Batch([1, 1], [700, 90], 16)                 # a table wide enough for a workspace
    cache = make_cache(batch, 2, 16, 64, E4M3)
    query = rows_like(2, 4, 64, torch.bfloat16, 1, 0.2)
    bad = query[:1].expand(2, 4, 64) if refused == "expanded rows" else query
    for _ in range(2):
        with pytest.raises(RuntimeError):
            cache.attention(bad, torch.zeros_like(query), *batch.meta, softmax_scale=1e-60 if refused == "scale" else None)
        check_attention(cache, batch, query)
