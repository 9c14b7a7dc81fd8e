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
All three read any positive finite scales and finite codes (`append` keeps a block's scale, whatever it is, where it is large enough).

Nothing here but `attention_status` synchronizes, and every other call can be captured in a CUDA graph.  Calls go to the current
stream of the cache's device; scratch memory is taken from PyTorch's allocator for each call, so calls on different streams share
none.  Rejected arguments raise RuntimeError.
"""

from __future__ import annotations

import struct
from typing import Optional, Tuple

import torch

from . import _lib
from ._cuda import _require

__all__ = ("BlockCache",)

_ELEMENTS = {torch.float8_e4m3fn: 0, torch.int8: 1}
_ACTIVATIONS = {torch.bfloat16: 0, torch.float16: 1}

# A decode step issues these calls once for each layer, so the argument structures of include/rq_b200.h are packed in one go
# (a tenth of what filling them field by field takes).
_CACHE, _BATCH = "PPPqiiii", "PPPiii4x"
_APPEND = struct.Struct("@" + _CACHE + _BATCH + "PPqqiiPi4x")
_ATTENTION = struct.Struct("@" + _CACHE + _BATCH + "PPqqiiiif4xPi4xPNPi4x")
_EVICT = struct.Struct("@" + _CACHE + _BATCH + "iii4xPPPi4x")


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
        self._view = (codes.data_ptr(), scales.data_ptr(), weights.data_ptr() if weights is not None else 0,
                      blocks, heads, head_dim, block_size, _ELEMENTS[codes.dtype])
        self._workspaces = {}   # bytes that an attention call of some sizes needs

    @classmethod
    def allocate(cls, num_blocks: int, kv_heads: int, head_dim: int, block_size: int = 16, dtype: torch.dtype = torch.float8_e4m3fn,
                 weights: bool = False, device="cuda") -> "BlockCache":
        """A zeroed cache of `num_blocks` blocks; `weights` adds the accumulated attention weights."""
        codes = torch.zeros(2, num_blocks, kv_heads, block_size, head_dim, dtype=torch.uint8, device=device).view(dtype)
        scales = torch.ones(2, num_blocks, kv_heads, device=device)
        return cls(codes, scales, torch.zeros(num_blocks, kv_heads, block_size, device=device) if weights else None)

    def _batch(self, query_start_loc, seq_lens, block_table) -> tuple:
        device = self.device
        if not (seq_lens.device == device and seq_lens.dtype == torch.int32 and seq_lens.dim() == 1 and seq_lens.is_contiguous()):
            raise RuntimeError("Contiguous INT32 sequence lengths required")
        requests = seq_lens.numel()
        starts = 0
        if query_start_loc is not None:
            if not (query_start_loc.device == device and query_start_loc.dtype == torch.int32 and query_start_loc.dim() == 1
                    and query_start_loc.is_contiguous() and query_start_loc.numel() == requests + 1):
                raise RuntimeError("Contiguous INT32 query starts with one final boundary required")
            starts = query_start_loc.data_ptr()
        if not (block_table.device == device and block_table.dtype == torch.int32 and block_table.dim() == 2):
            raise RuntimeError("INT32 page table with packed rows required")
        rows, width = block_table.shape
        row_stride, stride = block_table.stride()
        if not ((stride == 1 or width <= 1) and rows >= requests and (row_stride >= width or rows <= 1)):
            raise RuntimeError("INT32 page table with packed rows required")
        return starts, seq_lens.data_ptr(), block_table.data_ptr(), requests, max(row_stride, width), width

    def _rows(self, t: torch.Tensor, heads: int, what: str) -> int:
        """The stride between the rows of [rows, heads, head dim]."""
        if t.device == self.device and t.dtype in _ACTIVATIONS and t.dim() == 3:
            _, own_heads, dim = t.shape
            stride, head_stride, unit = t.stride()
            if own_heads == heads and dim == self.head_dim and unit == 1 and (heads == 1 or head_stride == dim):
                return stride
        raise RuntimeError(f"BF16 or FP16 [tokens, {heads}, {self.head_dim}] {what} with packed trailing strides on the cache device required")

    def _stream(self) -> int:
        return torch._C._cuda_getCurrentRawStream(self.device.index)

    def _on_device(self, function, args: bytes) -> int:
        if torch.cuda.current_device() == self.device.index:
            return function(args)
        with torch.cuda.device(self.device.index):
            return function(args)

    def _call(self, function, args: bytes) -> None:
        status = self._on_device(function, args)
        if status != _lib.RQ_OK:
            _lib.check(status)

    def append(self, key: torch.Tensor, value: torch.Tensor, query_start_loc: torch.Tensor, seq_lens: torch.Tensor,
               block_table: torch.Tensor) -> None:
        """Quantize the step's K/V rows [rows, kv heads, head dim] into their blocks.

        A block that the call begins (its slot 0 is written) takes the scale of its new tokens; a block that held earlier
        tokens of the request keeps its scale or, where the new tokens need a larger one, takes that and has the earlier
        tokens rounded again.  The new tokens' accumulated weights start at 0."""
        key_stride, value_stride = self._rows(key, self.kv_heads, "key"), self._rows(value, self.kv_heads, "value")
        rows = key.size(0)
        if key.dtype != value.dtype or value.size(0) != rows:
            raise RuntimeError("K and V must match in type and row count")
        batch = self._batch(query_start_loc, seq_lens, block_table)
        if rows and batch[3]:
            row = self.kv_heads * self.head_dim
            self._call(self._lib.rq_block_append, _APPEND.pack(
                *self._view, *batch, key.data_ptr(), value.data_ptr(), key_stride if rows > 1 else row, value_stride if rows > 1 else row,
                rows, _ACTIVATIONS[key.dtype], self._stream(), 0))

    def attention(self, query: torch.Tensor, output: torch.Tensor, query_start_loc: torch.Tensor, seq_lens: torch.Tensor,
                  block_table: torch.Tensor, *, softmax_scale: Optional[float] = None, lse: Optional[torch.Tensor] = None,
                  accumulate: bool = False, max_seq_len: Optional[int] = None) -> None:
        """Softmax attention of the step's rows [rows, heads, head dim] over the cached tokens, the step's own included (`append`
        them first); writes `output` in place, and the natural logarithm of the softmax denominators into `lse`
        [rows, heads] fp32.  `heads` is a multiple of the cache's heads; query head h reads KV head h // (heads // kv heads).
        `softmax_scale` defaults to head_dim ** -0.5.  Rows that see no token get zeros and -inf; padding rows stay as they are.

        `accumulate` adds every token's softmax weight, summed over the rows and over the query heads of its KV head, to the
        cache's `weights`.  Such a call needs scratch memory for rows x heads x `max_seq_len` scores.  `max_seq_len` (default: the
        block table's width) must be no smaller than any of `seq_lens`: tokens behind it are not seen; up to 512 saves a launch."""
        heads = query.size(1) if query.dim() == 3 else 0
        query_stride, output_stride = self._rows(query, heads, "query"), self._rows(output, heads, "output")
        rows = query.size(0)
        if output.dtype != query.dtype or output.size(0) != rows:
            raise RuntimeError("Q and output must match in type and row count")
        if heads == 0 or heads % self.kv_heads:
            raise RuntimeError(f"{heads} query heads are no multiple of the cache's {self.kv_heads} heads")
        if rows <= 1:
            query_stride = output_stride = heads * self.head_dim
        query_address, output_address = query.data_ptr(), output.data_ptr()
        if (query_address | output_address) % 16 or (query_stride | output_stride) % 8:
            raise RuntimeError("Q/output addresses and token strides must be 16-byte aligned")
        if lse is not None and not (lse.device == self.device and lse.dtype == torch.float32 and lse.is_contiguous()
                                    and lse.shape == (rows, heads)):
            raise RuntimeError("Contiguous FP32 [tokens, heads] lse required")
        if accumulate and self.weights is None:
            raise RuntimeError("accumulating needs a cache with weights")
        if max_seq_len is not None and max_seq_len <= 0:
            raise RuntimeError("max_seq_len must be positive")
        batch = self._batch(query_start_loc, seq_lens, block_table)
        if not rows or not batch[3]:
            return
        scale = self.head_dim ** -0.5 if softmax_scale is None else softmax_scale
        if not 0.0 < scale < 1e30:
            raise RuntimeError("softmax scale must be positive and finite")
        front = (*self._view, *batch, query_address, output_address, query_stride, output_stride, rows, heads, _ACTIVATIONS[query.dtype],
                 bool(accumulate), scale, lse.data_ptr() if lse is not None else 0, min(max_seq_len or 0, 0x7FFFFFFF))
        sizes = (rows, heads, batch[3], batch[5], bool(accumulate), max_seq_len)
        known = self._workspaces.get(sizes)
        nbytes = known
        if known is None:  # (it depends on the device's size too)
            nbytes = self._on_device(self._lib.rq_block_attention_workspace_bytes, _ATTENTION.pack(*front, 0, 0, 0, 0))
        workspace = self.codes.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        self._call(self._lib.rq_block_attention,
                   _ATTENTION.pack(*front, workspace.data_ptr() if nbytes else 0, nbytes, self._stream(), 0))
        if known is None:  # only now: of arguments that the call refuses the size is 0
            if len(self._workspaces) >= 4096:
                self._workspaces.clear()
            self._workspaces[sizes] = nbytes

    def attention_status(self) -> None:
        """Synchronize and raise if a bounded wait inside an attention kernel of any block cache ever gave up on this device."""
        with torch.cuda.device(self.device):
            _lib.check(self._lib.rq_block_attention_status(torch.cuda.current_stream().cuda_stream))

    def evict(self, seq_lens: torch.Tensor, block_table: torch.Tensor, budget: int, *, sinks: int = 0, recent: int = 0,
              kept: Optional[torch.Tensor] = None, new_lens: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Bring every request of more than `budget` tokens down to `budget`, for each KV head on its own: the first `sinks` tokens,
        the last `recent` ones and those of the others with the largest accumulated weight (ties: the lowest position, NaN
        last) move, in their order, to the first `budget` positions of the request's blocks, with their weights.  Requests of at
        most `budget` tokens are left alone.  This cache no longer needs the blocks behind ceil(budget / block size); owners that share
        the block table and are not evicted with it do, and keep their own lengths.

        Returns `kept` int32 [requests, kv heads, budget], the positions that the tokens now at 0, 1, ... had before (-1 behind
        the last), and `new_lens` int32 [requests], min(seq_len, budget); both can be passed in (not `seq_lens` itself)."""
        if self.weights is None:
            raise RuntimeError("evicting needs a cache with weights")
        if not (1 <= budget < 1 << 24 and sinks >= 0 and recent >= 0 and sinks + recent <= budget):
            raise RuntimeError(f"A budget of {budget} tokens cannot hold the first {sinks} and the last {recent}")
        batch = self._batch(None, seq_lens, block_table)
        requests = batch[3]
        if kept is None:
            kept = torch.empty(requests, self.kv_heads, budget, dtype=torch.int32, device=self.device)
        elif not (kept.device == self.device and kept.dtype == torch.int32 and kept.is_contiguous()
                  and kept.shape == (requests, self.kv_heads, budget)):
            raise RuntimeError("Contiguous INT32 [requests, heads, budget] kept positions required")
        if new_lens is None:
            new_lens = torch.empty(requests, dtype=torch.int32, device=self.device)
        elif not (new_lens.device == self.device and new_lens.dtype == torch.int32 and new_lens.is_contiguous()
                  and new_lens.shape == (requests,)):
            raise RuntimeError("Contiguous INT32 [requests] new lengths required")
        if requests:
            if abs(new_lens.data_ptr() - batch[1]) < 4 * requests:
                raise RuntimeError("new_lens must not share memory with seq_lens")
            self._call(self._lib.rq_block_evict, _EVICT.pack(
                *self._view, *batch, budget, sinks, recent, kept.data_ptr(), new_lens.data_ptr(), self._stream(), 0))
        return kept, new_lens
