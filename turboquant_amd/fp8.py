"""A paged cache in 8 bits: keys and values in e4m3 with a power of two for every block of 16 tokens and KV head.

It stands between the engine's exact blocks and `PagedKVPool`'s pages of two to four bits: half the exact cache's bytes, every value within 2^-4 of itself
(as long as it is not some thousand times smaller than its block's largest).  Its blocks and tables are the engine's, like those of
`ExactPagedCache`, and it answers the same calls: single tokens, several rows of a sequence, whole prompts, within a window or without.
(New: the reference quantises by rotation and codebook only, store.py.)
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _ffi
from .attend import HEAD_DIMS, attend, overlaps, plan_bytes, row_strides, seen_by, sequences, step_starts
from .eviction import own_rows
from .paged import PAGE_TOKENS


class Fp8PagedCache:
    """Key and value blocks (num_blocks, 16, H_kv, d) in torch.float8_e4m3fn, equal strides, channels contiguous, rows on 16-byte boundaries, and their
    scales (num_blocks, H_kv) uint8, contiguous: the byte e + 127 says that the block's elements of that KV head stand for 2^e times themselves.  The object
    holds the four tensors and nothing else; head_dim 64, 128, 192 or 256."""

    dtype = torch.float8_e4m3fn
    _tag = _ffi.TQ_E4M3

    def __init__(self, key_cache: torch.Tensor, value_cache: torch.Tensor, key_scales: torch.Tensor, value_scales: torch.Tensor):
        self.key_cache, self.value_cache, self.key_scales, self.value_scales = key_cache, value_cache, key_scales, value_scales
        fast = _ffi.native()
        known = None if fast is None else fast.fp8_cache(key_cache, value_cache, key_scales, value_scales)
        if known is not None:
            self.num_blocks, self.num_kv_heads, self.head_dim, self._strides = known
            self.device = key_cache.device
            return
        for name, t in self.tensors().items():
            _ffi.require_gpu(t, name)
        if key_cache.dim() != 4 or key_cache.shape != value_cache.shape or key_cache.shape[1] != PAGE_TOKENS:
            raise ValueError("key_cache and value_cache must both be (num_blocks, 16, H, d)")
        self.device = key_cache.device
        if any(t.dtype != torch.float8_e4m3fn for t in (key_cache, value_cache)) or any(t.dtype != torch.uint8 for t in (key_scales, value_scales)):
            raise TypeError("key_cache and value_cache must be float8_e4m3fn, key_scales and value_scales uint8")
        if any(t.is_neg() or t._is_zerotensor() for t in self.operands()):
            raise ValueError("the cache must hold its values: a lazily negated tensor does not")
        if any(t.device != self.device for t in (value_cache, key_scales, value_scales)):
            raise TypeError("the cache and its scales must live on one GPU")
        self.num_blocks, _, self.num_kv_heads, self.head_dim = key_cache.shape
        if self.head_dim not in HEAD_DIMS or self.num_kv_heads == 0 or self.num_blocks == 0:
            raise ValueError(f"head_dim must be one of {', '.join(map(str, HEAD_DIMS))}, got a cache of shape {tuple(key_cache.shape)}")
        if any(t.shape != (self.num_blocks, self.num_kv_heads) or not t.is_contiguous() for t in (key_scales, value_scales)):
            raise ValueError(f"key_scales and value_scales must be contiguous ({self.num_blocks}, {self.num_kv_heads})")
        self._strides = key_cache.stride()
        if (value_cache.stride() != self._strides or self._strides[3] != 1 or any(s % 16 for s in self._strides[:3]) or
                self._strides[1] > 1 << 24 or key_cache.data_ptr() % 16 or value_cache.data_ptr() % 16):
            raise ValueError("key_cache and value_cache need the same strides, contiguous channels and rows on 16-byte boundaries")

    @classmethod
    def allocate(cls, num_blocks: int, num_kv_heads: int, head_dim: int, device) -> "Fp8PagedCache":
        """A cache of its own, all zeros."""
        shape = (num_blocks, PAGE_TOKENS, num_kv_heads, head_dim)
        blocks = [torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2)]
        return cls(*blocks, *(torch.zeros(shape[0], shape[2], dtype=torch.uint8, device=device) for _ in range(2)))

    def tensors(self) -> dict:
        return dict(key_cache=self.key_cache, value_cache=self.value_cache, key_scales=self.key_scales, value_scales=self.value_scales)

    def operands(self):
        return self.key_cache, self.value_cache, self.key_scales, self.value_scales

    def _memory(self):
        return tuple(t.data_ptr() for t in self.operands())

    def memory_bytes(self) -> int:
        return sum(t.numel() for t in self.tensors().values())

    # ---- write and read back ---------------------------------------------------------------------------------------------
    def write(self, key: torch.Tensor, value: torch.Tensor, query_start_loc: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor) -> None:
        """Quantise a step's keys and values (rows, H_kv, d), fp32, fp16 or bf16, into the blocks of their tokens: row i of sequence b's
        n = query_start_loc[b + 1] - query_start_loc[b] is token seq_lens[b] - n + i, in block block_table[b][token // 16].

        A block's scale is the smallest power of two that brings its largest finite value to 448 at most; infinite values become the largest that
        it holds, NaN stays.  Tokens that a block holds already are rounded again where a new one needs a larger scale; a block whose first slot is written
        starts anew.  (A sequence that steps back behind a refused token and writes another in its place keeps the scale that it had raised, and the bits that the block's
        earlier tokens lost by it.)  A sequence's blocks must be its own while it writes to them; rows in front of token 0, behind the table or in blocks outside
        the cache are left out."""
        fast = _ffi.native()
        if fast is not None and fast.fp8_write(key, value, query_start_loc, block_table, seq_lens, *self.operands()):
            return
        _ffi.require_gpu(key, "key")
        _ffi.require_gpu(value, "value")
        if key.dim() != 3 or key.shape != value.shape or tuple(key.shape[1:]) != (self.num_kv_heads, self.head_dim):
            raise ValueError(f"key and value must both be (rows, {self.num_kv_heads}, {self.head_dim})")
        tag = _ffi.dtype_tag(key.dtype)
        if value.dtype != key.dtype or key.device != self.device or value.device != self.device:
            raise TypeError("key and value must have one dtype and live on the cache's GPU")
        _ffi.require_constant("write", key=key, value=value, **self.tensors())
        if any(overlaps(t, held) for t in (key, value) for held in self.tensors().values()):
            raise ValueError("key and value must not lie in the cache's own memory")
        k, v, k_scales, v_scales = self.operands()
        if not own_rows(k, v) or overlaps(k_scales, v_scales) or any(overlaps(x, y) for x in (k, v) for y in (k_scales, v_scales)):
            raise ValueError("a cache that overlaps itself cannot be written to")
        starts, B = step_starts(self.device, query_start_loc)
        table, bt_stride, lens = sequences(self.device, block_table, seq_lens, B)
        if bt_stride < 0 and B > 1:
            raise ValueError(f"one table for {B} sequences: they would write to the same blocks")
        if any(overlaps(t, held) for t in (starts, table, lens) for held in self.tensors().values()):
            raise ValueError("query_start_loc, block_table and seq_lens must not lie in the cache's own memory")
        rows = key.shape[0]
        if rows == 0 or B == 0:
            return
        key, value = (self._rows_of(t) for t in (key, value))
        with _ffi.on_device(self.device):
            _ffi.check(_ffi.lib().tq_fp8_write(
                key.data_ptr(), value.data_ptr(), tag, rows, *row_strides(key), *row_strides(value), starts.data_ptr(), B, self.num_kv_heads,
                self.head_dim, *self._memory(), *self._strides[:3], self.num_blocks, table.data_ptr(), bt_stride, lens.data_ptr(),
                _ffi.stream_ptr(self.device)), "tq_fp8_write")
        _ffi.changed(*self.tensors().values())

    @staticmethod
    def _rows_of(t: torch.Tensor) -> torch.Tensor:
        """Rows as the library reads them: channels contiguous, on 16-byte boundaries."""
        t = t.resolve_neg()
        piece = 16 // t.element_size()
        if t.stride(2) != 1 or any(s % piece for s in row_strides(t)) or t.data_ptr() % 16:
            t = t.contiguous()
            if t.data_ptr() % 16:
                t = t.clone()
        return t

    def read(self, query_start_loc: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, rows: Optional[int] = None,
             dtype: torch.dtype = torch.bfloat16, out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """What is held of the tokens that `write` takes the same arguments for: keys and values (rows, H_kv, d), each rounded once to `dtype`.
        rows: query_start_loc's last entry, which the host does not know.  A row whose token is not in the cache is zeros, and so are
        rows behind the last sequence; with out=(keys, values), contiguous, those are left as they are."""
        fast = _ffi.native()
        if fast is not None and out is None and rows is not None:
            done = fast.fp8_read(query_start_loc, block_table, seq_lens, rows, _ffi.dtype_tag(dtype), *self.operands())
            if done is not None:
                return done
        starts, B = step_starts(self.device, query_start_loc)
        table, bt_stride, lens = sequences(self.device, block_table, seq_lens, B)
        shape = (self.num_kv_heads, self.head_dim)
        if out is None:
            if rows is None or rows < 0:
                raise ValueError("read needs the number of rows, or out")
            _ffi.dtype_tag(dtype)
            keys, values = (torch.empty(rows, *shape, dtype=dtype, device=self.device) for _ in range(2))
        else:
            keys, values = out
            for t in out:
                if (t.dim() != 3 or t.shape != keys.shape or tuple(t.shape[1:]) != shape or (rows is not None and t.shape[0] != rows) or t.dtype != keys.dtype or
                        t.device != self.device or not t.is_contiguous() or t.is_neg() or t.data_ptr() % 16):
                    raise ValueError(f"out must be two contiguous tensors ({'rows' if rows is None else rows}, {shape[0]}, {shape[1]}) of one dtype on the cache's GPU")
                if any(overlaps(t, o) for o in self.tensors().values()):
                    raise ValueError("out must not lie in the cache's own memory")
            if any(overlaps(t, o) for t in out for o in (starts, table, lens)):
                raise ValueError("out must not lie over query_start_loc, block_table or seq_lens")
            if overlaps(keys, values):
                raise ValueError("the two tensors of out must not overlap")
        _ffi.require_constant("read", keys=keys, values=values, **self.tensors())
        tag, rows = _ffi.dtype_tag(keys.dtype), keys.shape[0]
        if rows == 0:
            return keys, values
        with _ffi.on_device(self.device):
            _ffi.check(_ffi.lib().tq_fp8_read(
                keys.data_ptr(), values.data_ptr(), tag, rows, starts.data_ptr(), B, *shape, *self._memory(), *self._strides[:3],
                self.num_blocks, table.data_ptr(), bt_stride, lens.data_ptr(), int(out is None), _ffi.stream_ptr(self.device)), "tq_fp8_read")
        if out is not None:
            _ffi.changed(keys, values)
        return keys, values

    # ---- attention -----------------------------------------------------------------------------------------------------------
    def decode_attention(self, query: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, scale: Optional[float] = None,
                         window: Optional[int] = None, sinks: int = 0, n_split: Optional[int] = None, workspace: Optional[torch.Tensor] = None,
                         out: Optional[torch.Tensor] = None, max_len: Optional[int] = None) -> torch.Tensor:
        """`attention` of one row per sequence, its newest token: query (B, Hq, d), fp16 or bf16."""
        return attend("decode_attention", self, query, None, block_table, seq_lens, scale, window, sinks, n_split, workspace, out, max_len, None)

    def attention(self, query: torch.Tensor, query_start_loc: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                  scale: Optional[float] = None, window: Optional[int] = None, sinks: int = 0, n_split: Optional[int] = None,
                  workspace: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, max_len: Optional[int] = None,
                  max_rows: Optional[int] = None) -> torch.Tensor:
        """softmax(scale * q K^T) V for the rows of a step, query (rows, Hq, d) in fp16 or bf16, whose keys and values are written: row i of sequence b's n
        stands at position p = seq_lens[b] - n + i and sees the tokens up to its own; with a window only those behind p - window, and the first
        `sinks`.  A row that sees nothing is zeros.  Rows behind the last sequence are zeros, or left as they are in a given `out`.

        max_len and max_rows bound the lengths and a sequence's rows for the plan of the splits (without them the table's width and all rows
        do).  Of up to 32 rows x heads on a KV head, in decode steps and for fp16 queries the softmax's weights go into the product with the values as two
        numbers of 16 bits, 2^-15 of a weight off, otherwise as one of the query's type, half a step off.  The `workspace` of a step (`workspace()` of the
        same sizes and bounds) belongs to it alone until it has run: graphs that may run at the same time need one each."""
        return attend("attention", self, query, query_start_loc, block_table, seq_lens, scale, window, sinks, n_split, workspace, out, max_len, max_rows)

    def workspace(self, rows: int, Hq: int, max_len: int, B: Optional[int] = None, max_rows: Optional[int] = None, window: Optional[int] = None,
                  sinks: int = 0, n_split: Optional[int] = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """A workspace for steps of this size: `attention` of B sequences, or, without B, `decode_attention`."""
        window, sinks = seen_by(window, sinks)
        need = plan_bytes(self, dtype, B is not None, rows, rows if B is None else B, Hq, max_len, rows if max_rows is None else max_rows, window, sinks,
                          n_split or 0)
        return torch.empty(need // 4, dtype=torch.float32, device=self.device)
