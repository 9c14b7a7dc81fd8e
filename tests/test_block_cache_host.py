"""Refusals and sizes of the block cache's C ABI, and the cache class without a GPU (CPU)."""

import ctypes

import pytest
import torch

from residualquant_b200 import _lib, block_cache
from residualquant_b200.block_cache import BlockCache

ADDRESS = 1 << 20   # a pointer that is only looked at


def append_args(**changes):
    cache = dict(codes=ADDRESS, scales=ADDRESS, weights=ADDRESS, num_blocks=8, kv_heads=2, head_dim=128, page_tokens=16, element=0)
    batch = dict(query_start_loc=ADDRESS, seq_lens=ADDRESS, block_table=ADDRESS, num_requests=2, block_table_stride=4, max_blocks_per_request=4)
    rest = dict(key=ADDRESS, value=ADDRESS, key_stride=256, value_stride=256, num_rows=0, activation=0)
    return _fill(_lib.RqBlockAppendArgs, cache, batch, rest, changes)


def attention_args(**changes):
    cache = dict(codes=ADDRESS, scales=ADDRESS, weights=ADDRESS, num_blocks=8, kv_heads=2, head_dim=128, page_tokens=16, element=0)
    batch = dict(query_start_loc=ADDRESS, seq_lens=ADDRESS, block_table=ADDRESS, num_requests=2, block_table_stride=4, max_blocks_per_request=4)
    rest = dict(query=ADDRESS, output=ADDRESS, query_stride=1024, output_stride=1024, num_rows=3, heads=8, activation=0, accumulate=0,
                softmax_scale=0.1)
    return _fill(_lib.RqBlockAttentionArgs, cache, batch, rest, changes)


def evict_args(**changes):
    cache = dict(codes=ADDRESS, scales=ADDRESS, weights=ADDRESS, num_blocks=8, kv_heads=2, head_dim=128, page_tokens=16, element=0)
    batch = dict(query_start_loc=None, seq_lens=ADDRESS, block_table=ADDRESS, num_requests=2, block_table_stride=4, max_blocks_per_request=4)
    return _fill(_lib.RqBlockEvictArgs, cache, batch, dict(budget=0, sinks=0, recent=0, kept=ADDRESS, new_lens=None), changes)


def _fill(kind, cache, batch, rest, changes):
    for part in (cache, batch, rest):
        part.update({k: v for k, v in changes.items() if k in part})
    return kind(cache=_lib.RqBlockCache(**cache), batch=_lib.RqBlockBatch(**batch), **rest)


BAD_CACHE = [dict(head_dim=80), dict(page_tokens=24), dict(element=2), dict(kv_heads=0), dict(num_blocks=0), dict(codes=None),
             dict(codes=ADDRESS + 8), dict(scales=None), dict(num_requests=0), dict(seq_lens=None), dict(block_table=None),
             dict(block_table_stride=3), dict(max_blocks_per_request=-1), dict(num_blocks=1 << 40)]


@pytest.mark.parametrize("changes", BAD_CACHE + [dict(query_start_loc=None), dict(num_rows=-1)])
def test_append_refuses(built_library, changes):
    lib = _lib.load()
    assert lib.rq_block_append(ctypes.byref(append_args())) == 0           # nothing to do, nothing launched
    assert lib.rq_block_append(ctypes.byref(append_args(**changes))) < 0
    assert lib.rq_last_error()


@pytest.mark.parametrize("changes", [dict(key=None), dict(value=ADDRESS + 1), dict(key_stride=255), dict(activation=7),
                                     dict(num_rows=0x7FFFFFFF)])
def test_append_refuses_rows(built_library, changes):
    lib = _lib.load()
    assert lib.rq_block_append(ctypes.byref(append_args(**{"num_rows": 1, **changes}))) < 0
    assert lib.rq_block_append(None) == -1


@pytest.mark.parametrize("changes", BAD_CACHE + [
    dict(query_start_loc=None), dict(heads=3), dict(heads=0), dict(query=None), dict(output=ADDRESS + 8), dict(query_stride=1023),
    dict(output_stride=1028), dict(softmax_scale=0.0), dict(softmax_scale=float("nan")), dict(softmax_scale=float("inf")),
    dict(activation=2), dict(num_rows=-1), dict(num_rows=1 << 28), dict(accumulate=1, weights=None)])
def test_attention_refuses(built_library, changes):
    lib = _lib.load()
    args = attention_args(**changes)
    assert lib.rq_block_attention(ctypes.byref(args)) < 0
    assert lib.rq_block_attention_workspace_bytes(ctypes.byref(args)) == 0
    assert lib.rq_block_attention(None) == -1 and lib.rq_block_attention_workspace_bytes(None) == 0


def test_attention_asks_for_its_workspace(built_library):
    lib = _lib.load()
    wide = dict(block_table_stride=100, max_blocks_per_request=100)
    args = attention_args(**wide)
    need = lib.rq_block_attention_workspace_bytes(ctypes.byref(args))
    assert need > 0 and need % 256 == 0
    assert lib.rq_block_attention(ctypes.byref(args)) == -3                 # none given
    args.workspace, args.workspace_bytes = ADDRESS, need - 1
    assert lib.rq_block_attention(ctypes.byref(args)) == -3
    args.workspace, args.workspace_bytes = ADDRESS + 16, need
    assert lib.rq_block_attention(ctypes.byref(args)) == -3
    assert lib.rq_block_attention(ctypes.byref(attention_args(num_rows=0))) == 0
    # the scores and denominators of an accumulating call: rows x heads x the length bound
    counted = lib.rq_block_attention_workspace_bytes(ctypes.byref(attention_args(accumulate=1, **wide)))
    assert counted == need + 256 + 3 * 8 * 1600 * 4
    # short tables: no item is cut, so only what is accumulated
    assert lib.rq_block_attention_workspace_bytes(ctypes.byref(attention_args())) == 0
    assert lib.rq_block_attention_workspace_bytes(ctypes.byref(attention_args(accumulate=1))) == 256 + 3 * 8 * 64 * 4


@pytest.mark.parametrize("changes", BAD_CACHE + [dict(weights=None), dict(), dict(budget=4, sinks=3, recent=2), dict(budget=4, sinks=-1),
                                                 dict(budget=4, recent=-1), dict(budget=4, kept=None), dict(budget=4, kept=ADDRESS + 2),
                                                 dict(budget=4, new_lens=ADDRESS), dict(budget=1 << 30)])
def test_evict_refuses(built_library, changes):
    lib = _lib.load()
    if changes in BAD_CACHE:
        changes = dict(budget=4, **changes)
    assert lib.rq_block_evict(ctypes.byref(evict_args(**changes))) < 0
    assert lib.rq_block_evict(None) == -1


def test_packed_arguments_have_the_layout_of_the_structures():
    for packed, kind in ((block_cache._APPEND, _lib.RqBlockAppendArgs), (block_cache._ATTENTION, _lib.RqBlockAttentionArgs),
                         (block_cache._EVICT, _lib.RqBlockEvictArgs)):
        assert packed.size == ctypes.sizeof(kind)
        flat = []
        for name, field in kind._fields_:
            inner = getattr(field, "_fields_", None)
            flat += [(name, n) for n, _ in inner] if inner else [(name,)]
        values = packed.pack(*range(1, len(flat) + 1))          # a whole number for every field, the float among them
        args = kind.from_buffer_copy(values)
        for i, path in enumerate(flat):
            field = getattr(args, path[0])
            assert (getattr(field, path[1]) if len(path) == 2 else field) == i + 1, path


def test_the_cache_lives_on_the_gpu(built_library):
    codes = torch.zeros(2, 4, 2, 16, 64, dtype=torch.int8)
    with pytest.raises(RuntimeError):
        BlockCache(codes, torch.ones(2, 4, 2))
    with pytest.raises(RuntimeError):
        BlockCache.allocate(4, 2, 64, device="cpu")


@pytest.mark.parametrize("page", [16, 32])
def test_a_table_of_more_than_2_to_the_30_tokens_is_refused(built_library, page):
    lib = _lib.load()
    most = (1 << 30) // page

    def table(pages):
        return dict(page_tokens=page, block_table_stride=pages, max_blocks_per_request=pages)

    assert 0 < lib.rq_block_attention_workspace_bytes(ctypes.byref(attention_args(**table(most)))) < 1 << 30
    assert lib.rq_block_append(ctypes.byref(append_args(**table(most)))) == 0                       # no rows
    for pages in (most + 1, 0x7FFFFFFF // page, 0x7FFFFFFF):
        assert lib.rq_block_attention_workspace_bytes(ctypes.byref(attention_args(**table(pages)))) == 0
        assert lib.rq_block_attention(ctypes.byref(attention_args(num_rows=0, **table(pages)))) == -1
        assert lib.rq_block_append(ctypes.byref(append_args(**table(pages)))) == -1
        assert lib.rq_block_evict(ctypes.byref(evict_args(budget=4, **table(pages)))) == -1


@pytest.mark.parametrize("offset,shared", [(-4, True), (0, True), (4, True), (4 * (1 << 30) - 4, True), (4 * (1 << 30), False)])
def test_new_lengths_that_share_memory_with_the_lengths_are_refused(built_library, offset, shared):
    lib = _lib.load()
    # 2^30 requests are too many in any case, so that nothing is launched; what is said first is the overlap
    assert lib.rq_block_evict(ctypes.byref(evict_args(budget=4, new_lens=ADDRESS + offset, num_requests=1 << 30))) == -1
    assert (b"seq_lens" in lib.rq_last_error()) == shared


@pytest.mark.parametrize("field", ["query_start_loc", "seq_lens", "block_table"])
def test_metadata_off_their_alignment_are_refused(built_library, field):
    lib = _lib.load()
    changes = {field: ADDRESS + 2}
    assert lib.rq_block_attention(ctypes.byref(attention_args(num_rows=0, **changes))) == -1
    assert lib.rq_block_append(ctypes.byref(append_args(**changes))) == -1
    if field != "query_start_loc":
        # (the second refusal keeps anything from being launched)
        assert lib.rq_block_evict(ctypes.byref(evict_args(budget=4, kept=ADDRESS + 2, **changes))) == -1
        assert b"kept" not in lib.rq_last_error()


def test_an_lse_off_its_alignment_is_refused(built_library):
    lib = _lib.load()
    args = attention_args(num_rows=0)
    args.lse = ADDRESS + 4
    assert lib.rq_block_attention(ctypes.byref(args)) == 0
    args.lse = ADDRESS + 2
    assert lib.rq_block_attention(ctypes.byref(args)) == -1


class HostCache(BlockCache):
    """A cache over CPU tensors whose attention calls end at the library's checks: `asked` are the workspace sizes that accepted calls
    came with, `devices` the devices that were current while the library was asked for sizes or called."""

    def __init__(self, monkeypatch, width):
        lib = _lib.load()
        self.codes, self.scales, self.weights = torch.zeros(2, 4, 2, 16, 64, dtype=torch.int8), torch.ones(2, 4, 2), None
        self.num_blocks, self.kv_heads, self.block_size, self.head_dim = 4, 2, 16, 64
        self.device, self._workspaces = self.codes.device, {}
        self._view = (self.codes.data_ptr(), self.scales.data_ptr(), 0, 4, 2, 64, 16, 1)
        self._lib, self.asked, self.devices = self, [], []
        self.batch = torch.tensor([0, 1]).int(), torch.tensor([5]).int(), torch.zeros(1, width, dtype=torch.int32)
        self.current = [7]                                     # not this cache's
        monkeypatch.setattr(torch.cuda, "current_device", lambda: self.current[-1])

        class Device:
            def __init__(device, index):
                device.index = index

            def __enter__(device):
                self.current.append(device.index)

            def __exit__(device, *_):
                self.current.pop()

        monkeypatch.setattr(torch.cuda, "device", Device)
        self.need = lib.rq_block_attention_workspace_bytes

    def _stream(self):
        return 0

    def rq_block_attention_workspace_bytes(self, args):
        self.devices.append(self.current[-1])
        return self.need(args)

    def rq_block_attention(self, args):
        self.devices.append(self.current[-1])
        given = _lib.RqBlockAttentionArgs.from_buffer_copy(args)
        need = self.need(args)
        if need == 0:
            return -1                                          # a table this wide needs one: the arguments are not valid
        self.asked.append((given.workspace_bytes, need))
        return 0


@pytest.mark.parametrize("refused", [dict(softmax_scale=1e-60), dict(expand=True)])
def test_a_refused_call_leaves_later_ones_alone(built_library, monkeypatch, refused):
    cache = HostCache(monkeypatch, 100)
    query = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    bad = query[:1].expand(2, 4, 64) if refused.get("expand") else query
    with pytest.raises(RuntimeError):
        cache.attention(bad, query, *cache.batch, softmax_scale=refused.get("softmax_scale"))
    for _ in range(2):
        cache.attention(query, query, *cache.batch)
    assert len(cache.asked) == 2 and all(given == need > 0 for given, need in cache.asked)


def test_the_workspace_is_sized_on_the_device_of_the_cache(built_library, monkeypatch):
    cache = HostCache(monkeypatch, 100)
    query = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    cache.attention(query, query, *cache.batch)
    assert cache.devices == [cache.device.index] * 2 and cache.current == [7]
