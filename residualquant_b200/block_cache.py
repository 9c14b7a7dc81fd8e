"""A paged KV cache held in 8 bits with one scale for each block of tokens and KV head, for KV owners that are not
residual-coded (the reference keeps those in bf16): what a layer appends, attends to and evicts.

    cache = BlockCache.allocate(num_blocks, kv_heads, head_dim, block_size=16, dtype=torch.float8_e4m3fn, weights=True)
    cache.append(key, value, query_start_loc, seq_lens, block_table)          # the step's K/V rows, first
    cache.attention(query, output, query_start_loc, seq_lens, block_table, accumulate=True)
    kept, new_lens = cache.evict(seq_lens, block_table, budget=2048, sinks=4, recent=256)

The metadata are those of `_cuda.attention`: int32 `query_start_loc` [requests + 1], `seq_lens` [requests] (the step's own tokens
included) and `block_table` [>= requests, blocks], all on the cache's device; rows behind query_start_loc[-1] are padding.  Row i
of a request's q rows stands at position seq_len - q + i and sees the positions up to its own.  No two requests of a call may
share a block that the call writes (`append`, `evict`; with `accumulate` shared blocks get the sum of both requests' weights, in
no fixed order).

A cached value is code * scale.  `append` and `evict` write scales that are powers of two: the smallest one that brings a block's
largest finite magnitude into the codes' range (448 for float8_e4m3fn, 127 for int8); infinities saturate and NaN is stored as 0.
`attention` reads any positive finite scales and finite codes.

Nothing here synchronizes, and every call can be captured in a CUDA graph.  Calls go to the current stream of the cache's device;
scratch memory is taken from PyTorch's allocator for each call, so calls on different streams share none.  Rejected arguments
raise RuntimeError.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib
from ._cuda import _require

__all__ = ("BlockCache",)

_ELEMENTS = {torch.float8_e4m3fn: 0, torch.int8: 1}
_ACTIVATIONS = {torch.bfloat16: 0, torch.float16: 1}


class BlockCache:
    """`codes` float8_e4m3fn or int8 [2, blocks, kv heads, block size, head dim] (plane 0 = K, plane 1 = V), `scales` fp32
    [2, blocks, kv heads] and, for `attention(accumulate=True)` and `evict`, `weights` fp32 [blocks, kv heads, block size]; all
    contiguous.  The tensors stay the caller's: their contents may be read and written between calls."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, weights: Optional[torch.Tensor] = None) -> None:
        _require(
            codes.is_cuda and codes.dtype in _ELEMENTS and codes.dim() == 5 and codes.size(0) == 2 and codes.is_contiguous()
            and codes.data_ptr() % 16 == 0,
            "Contiguous CUDA FLOAT8_E4M3FN or INT8 [2, blocks, heads, block size, channels] codes required",
        )
        _, blocks, heads, block_size, head_dim = codes.shape
        _require(head_dim in (64, 96, 128) and block_size in (16, 32) and blocks > 0 and heads > 0,
                 f"No block-cache kernel for {heads} heads of {head_dim} channels in {blocks} blocks of {block_size} tokens")
        _require(
            scales.device == codes.device and scales.dtype == torch.float32 and scales.is_contiguous()
            and tuple(scales.shape) == (2, blocks, heads),
            "Contiguous FP32 [2, blocks, heads] scales on the codes' device required",
        )
        _require(
            weights is None
            or (weights.device == codes.device and weights.dtype == torch.float32 and weights.is_contiguous()
                and weights.data_ptr() % 16 == 0 and tuple(weights.shape) == (blocks, heads, block_size)),
            "Contiguous FP32 [blocks, heads, block size] weights on the codes' device required",
        )
        self.codes, self.scales, self.weights = codes, scales, weights
        self.num_blocks, self.kv_heads, self.block_size, self.head_dim = blocks, heads, block_size, head_dim
        self.device = codes.device
        self._lib = _lib.load()
        self._view = _lib.RqBlockCache(codes.data_ptr(), scales.data_ptr(), weights.data_ptr() if weights is not None else None,
                                       blocks, heads, head_dim, block_size, _ELEMENTS[codes.dtype])

    @classmethod
    def allocate(cls, num_blocks: int, kv_heads: int, head_dim: int, block_size: int = 16, dtype: torch.dtype = torch.float8_e4m3fn,
                 weights: bool = False, device="cuda") -> "BlockCache":
        """A zeroed cache of `num_blocks` blocks; `weights` adds the accumulated attention weights."""
        codes = torch.zeros(2, num_blocks, kv_heads, block_size, head_dim, dtype=torch.uint8, device=device).view(dtype)
        scales = torch.ones(2, num_blocks, kv_heads, device=device)
        return cls(codes, scales, torch.zeros(num_blocks, kv_heads, block_size, device=device) if weights else None)

    def _batch(self, query_start_loc, seq_lens, block_table) -> _lib.RqBlockBatch:
        device, requests = self.device, seq_lens.numel()
        _require(
            seq_lens.device == device and seq_lens.dtype == torch.int32 and seq_lens.dim() == 1 and seq_lens.is_contiguous(),
            "Contiguous INT32 sequence lengths required",
        )
        _require(
            query_start_loc is None
            or (query_start_loc.device == device and query_start_loc.dtype == torch.int32 and query_start_loc.dim() == 1
                and query_start_loc.is_contiguous() and query_start_loc.numel() == requests + 1),
            "Contiguous INT32 query starts with one final boundary required",
        )
        _require(
            block_table.device == device and block_table.dtype == torch.int32 and block_table.dim() == 2
            and (block_table.stride(1) == 1 or block_table.size(1) <= 1) and block_table.size(0) >= requests
            and block_table.stride(0) >= block_table.size(1),
            "INT32 page table with packed rows required",
        )
        return _lib.RqBlockBatch(query_start_loc.data_ptr() if query_start_loc is not None else None, seq_lens.data_ptr(),
                                 block_table.data_ptr(), requests, block_table.stride(0), block_table.size(1))

    def _rows(self, t: torch.Tensor, heads: int, what: str) -> None:
        _require(
            t.device == self.device and t.dtype in _ACTIVATIONS and t.dim() == 3 and t.size(1) == heads and t.size(2) == self.head_dim
            and t.stride(2) == 1 and (heads == 1 or t.stride(1) == self.head_dim),
            f"BF16 or FP16 [tokens, {heads}, {self.head_dim}] {what} with packed trailing strides on the cache device required",
        )

    def _call(self, function, args) -> None:
        index = self.device.index
        if torch.cuda.current_device() == index:
            args.stream = torch.cuda.current_stream(index).cuda_stream
            status = function(ctypes.byref(args))
        else:
            with torch.cuda.device(index):
                args.stream = torch.cuda.current_stream(index).cuda_stream
                status = function(ctypes.byref(args))
        if status != _lib.RQ_OK:
            _lib.check(status)

    def append(self, key: torch.Tensor, value: torch.Tensor, query_start_loc: torch.Tensor, seq_lens: torch.Tensor,
               block_table: torch.Tensor) -> None:
        """Quantize the step's K/V rows [rows, kv heads, head dim] into their blocks.

        A block that the call begins (its slot 0 is written) takes the scale of its new tokens; a block that held earlier
        tokens of the request keeps its scale or, where the new tokens need a larger one, takes that and has the earlier
        tokens rounded again.  The new tokens' accumulated weights start at 0."""
        for t, what in ((key, "key"), (value, "value")):
            self._rows(t, self.kv_heads, what)
        _require(key.dtype == value.dtype and key.size(0) == value.size(0), "K and V must match in type and row count")
        batch = self._batch(query_start_loc, seq_lens, block_table)
        if key.size(0) == 0 or seq_lens.numel() == 0:
            return
        args = _lib.RqBlockAppendArgs(self._view, batch, key.data_ptr(), value.data_ptr(), key.stride(0), value.stride(0),
                                      key.size(0), _ACTIVATIONS[key.dtype])
        self._call(self._lib.rq_block_append, args)

    def attention(self, query: torch.Tensor, output: torch.Tensor, query_start_loc: torch.Tensor, seq_lens: torch.Tensor,
                  block_table: torch.Tensor, *, softmax_scale: Optional[float] = None, lse: Optional[torch.Tensor] = None,
                  accumulate: bool = False, max_seq_len: Optional[int] = None) -> None:
        """Softmax attention of the step's rows [rows, heads, head dim] over the cached tokens, the step's own included (`append`
        them first); writes `output` in place, and the natural logarithm of the softmax denominators into `lse`
        [rows, heads] fp32.  `heads` is a multiple of the cache's heads; query head h reads KV head h // (heads // kv heads).
        `softmax_scale` defaults to head_dim ** -0.5.  Rows that see no token get zeros and -inf; padding rows stay as they are.

        `accumulate` adds every token's softmax weight, summed over the rows and over the query heads of its KV head, to the
        cache's `weights`.  Such a call needs scratch memory for rows x heads x `max_seq_len` scores; `max_seq_len` (default: the
        block table's width) must be no smaller than any of `seq_lens`: tokens behind it are not seen."""
        heads = query.size(1) if query.dim() == 3 else 0
        self._rows(query, heads, "query")
        self._rows(output, heads, "output")
        _require(output.dtype == query.dtype and output.size(0) == query.size(0), "Q and output must match in type and row count")
        _require(heads > 0 and heads % self.kv_heads == 0, f"{heads} query heads are no multiple of the cache's {self.kv_heads} heads")
        for t in (query, output):
            _require(t.data_ptr() % 16 == 0 and t.stride(0) % 8 == 0, "Q/output addresses and token strides must be 16-byte aligned")
        _require(
            lse is None
            or (lse.device == self.device and lse.dtype == torch.float32 and lse.is_contiguous()
                and tuple(lse.shape) == (query.size(0), heads)),
            "Contiguous FP32 [tokens, heads] lse required",
        )
        _require(not accumulate or self.weights is not None, "accumulating needs a cache with weights")
        _require(max_seq_len is None or max_seq_len > 0, "max_seq_len must be positive")
        batch = self._batch(query_start_loc, seq_lens, block_table)
        if query.size(0) == 0 or seq_lens.numel() == 0:
            return
        args = _lib.RqBlockAttentionArgs(
            self._view, batch, query.data_ptr(), output.data_ptr(), query.stride(0), output.stride(0), query.size(0), heads,
            _ACTIVATIONS[query.dtype], bool(accumulate), self.head_dim ** -0.5 if softmax_scale is None else softmax_scale,
            lse.data_ptr() if lse is not None else None, min(max_seq_len or 0, 0x7FFFFFFF))
        nbytes = self._lib.rq_block_attention_workspace_bytes(ctypes.byref(args))
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        args.workspace, args.workspace_bytes = workspace.data_ptr(), nbytes
        self._call(self._lib.rq_block_attention, args)

    def attention_status(self) -> None:
        """Synchronize and raise if a bounded wait inside an attention kernel of any block cache ever gave up on this device."""
        with torch.cuda.device(self.device):
            _lib.check(self._lib.rq_block_attention_status(torch.cuda.current_stream().cuda_stream))

    def evict(self, seq_lens: torch.Tensor, block_table: torch.Tensor, budget: int, *, sinks: int = 0, recent: int = 0,
              kept: Optional[torch.Tensor] = None, new_lens: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Bring every request of more than `budget` tokens down to `budget`, for each KV head on its own: the first `sinks` tokens,
        the last `recent` ones and those of the others with the largest accumulated weight (ties: the lowest position, NaN
        last) move, in their order, to the first `budget` positions of the request's blocks, with their weights.  Requests of at
        most `budget` tokens are left alone.  The blocks behind ceil(budget / block size) can be given back.

        Returns `kept` int32 [requests, kv heads, budget], the positions that the tokens now at 0, 1, ... had before (-1 behind
        the last), and `new_lens` int32 [requests], min(seq_len, budget); both can be passed in (not `seq_lens` itself)."""
        _require(self.weights is not None, "evicting needs a cache with weights")
        _require(budget >= 1 and sinks >= 0 and recent >= 0 and sinks + recent <= budget,
                 f"A budget of {budget} tokens cannot hold the first {sinks} and the last {recent}")
        batch = self._batch(None, seq_lens, block_table)
        requests = seq_lens.numel()
        if kept is None:
            kept = torch.empty(requests, self.kv_heads, budget, dtype=torch.int32, device=self.device)
        if new_lens is None:
            new_lens = torch.empty(requests, dtype=torch.int32, device=self.device)
        _require(
            kept.device == self.device and kept.dtype == torch.int32 and kept.is_contiguous()
            and tuple(kept.shape) == (requests, self.kv_heads, budget),
            "Contiguous INT32 [requests, heads, budget] kept positions required",
        )
        _require(
            new_lens.device == self.device and new_lens.dtype == torch.int32 and new_lens.is_contiguous()
            and tuple(new_lens.shape) == (requests,),
            "Contiguous INT32 [requests] new lengths required",
        )
        _require(abs(new_lens.data_ptr() - seq_lens.data_ptr()) >= 4 * requests or requests == 0,
                 "new_lens must not share memory with seq_lens")
        if requests:
            self._call(self._lib.rq_block_evict,
                       _lib.RqBlockEvictArgs(self._view, batch, budget, sinks, recent, kept.data_ptr(), new_lens.data_ptr()))
        return kept, new_lens
