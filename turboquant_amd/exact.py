"""Attention over the engine's paged exact cache, in place.

`PagedKVPool` answers decode steps from compressed pages; a layer that stays exact (the first ones, usually) or a sequence
that is not compressed yet is answered from the blocks that the engine keeps: (num_blocks, 16, H_kv, d) keys and values in
fp32, fp16 or bf16, reached through the same block tables.  Next to the attention itself every token's weight can be summed
per KV head, which is what `eviction.select_evictions` decides by.  (The reference leaves all of this to its engine's backend,
integration/vllm.py:290-318.)
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from . import _ffi
from .attend import attend, check_workspace, overlaps, plan_bytes, seen_by, sequences
from .eviction import Evictions, memory_of, own_rows
from .paged import PAGE_TOKENS

MAX_HEAD_DIM = 768
MAX_WINDOW = 1024


class ExactPagedCache:
    """An engine's key and value blocks, (num_blocks, 16, H_kv, d) each, equal strides, channels contiguous, rows on 16-byte
    boundaries; the object holds the two tensors and nothing else."""

    def __init__(self, key_cache: torch.Tensor, value_cache: torch.Tensor):
        self.key_cache, self.value_cache = key_cache, value_cache
        fast = _ffi.native()
        known = None if fast is None else fast.exact_cache(key_cache, value_cache)
        if known is not None:
            self._tag, self.num_blocks, self.num_kv_heads, self.head_dim, self._strides = known
            self.dtype, self.device = key_cache.dtype, key_cache.device
            return
        _ffi.require_gpu(key_cache, "key_cache")
        _ffi.require_gpu(value_cache, "value_cache")
        if key_cache.dim() != 4 or key_cache.shape != value_cache.shape or key_cache.shape[1] != PAGE_TOKENS:
            raise ValueError("key_cache and value_cache must both be (num_blocks, 16, H, d)")
        self.dtype, self.device = key_cache.dtype, key_cache.device
        self._tag = _ffi.dtype_tag(self.dtype)
        if value_cache.dtype != self.dtype or value_cache.device != self.device:
            raise TypeError("key_cache and value_cache must have one dtype and live on one GPU")
        self.num_blocks, _, self.num_kv_heads, self.head_dim = key_cache.shape
        if self.head_dim % 64 or not 0 < self.head_dim <= MAX_HEAD_DIM or self.num_kv_heads == 0 or self.num_blocks == 0:
            raise ValueError(f"head_dim must be a multiple of 64 up to {MAX_HEAD_DIM}, got a cache of shape {tuple(key_cache.shape)}")
        if any(t.is_neg() or t._is_zerotensor() for t in (key_cache, value_cache)):
            raise ValueError("key_cache and value_cache must hold their values: a lazily negated tensor does not")
        self._strides = key_cache.stride()
        piece = 16 // key_cache.element_size()
        if (value_cache.stride() != self._strides or self._strides[3] != 1 or any(s % piece for s in self._strides[:3]) or
                self._strides[1] > 1 << 24 or key_cache.data_ptr() % 16 or value_cache.data_ptr() % 16):
            raise ValueError("key_cache and value_cache need the same strides, contiguous channels and rows on 16-byte boundaries")

    @classmethod
    def from_engine(cls, kv_cache: torch.Tensor) -> "ExactPagedCache":
        """The cache of an attention module, (2, num_blocks, 16, H_kv, d)."""
        if kv_cache.dim() != 5 or kv_cache.shape[0] != 2:
            raise ValueError("expected (2, num_blocks, 16, H, d)")
        return cls(kv_cache[0], kv_cache[1])

    # ---- arguments that the calls share ------------------------------------------------------------------------------
    def _sequences(self, block_table: torch.Tensor, seq_lens: torch.Tensor, batch: int):
        """(table, its stride as the library takes it, lengths): int32 on this GPU, contiguous."""
        return sequences(self.device, block_table, seq_lens, batch)

    def _weights(self, weights: torch.Tensor, batch: int) -> None:
        _ffi.require_gpu(weights, "weights")
        if weights.dtype != torch.float32 or weights.device != self.device:
            raise TypeError("weights must be float32 on the cache's GPU")
        if weights.dim() != 3 or tuple(weights.shape[:2]) != (batch, self.num_kv_heads) or weights.shape[2] == 0:
            raise ValueError(f"weights must be ({batch}, {self.num_kv_heads}, tokens)")
        if weights.stride(2) != 1 or weights.is_neg():
            raise ValueError("weights need contiguous tokens, and memory that holds their values")
        if not own_rows(weights):
            raise ValueError("weights must not overlap themselves")

    # ---- read ----------------------------------------------------------------------------------------------------------
    def decode_attention(self, query: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                         scale: Optional[float] = None, weights: Optional[torch.Tensor] = None,
                         n_split: Optional[int] = None, workspace: Optional[torch.Tensor] = None,
                         out: Optional[torch.Tensor] = None, max_len: Optional[int] = None, window: Optional[int] = None,
                         sinks: int = 0) -> torch.Tensor:
        """softmax(scale * q K^T) V for one query token per sequence, query (B, Hq, d) in the cache's dtype, over the
        seq_lens[b] tokens that block_table (B, max_pages) or (max_pages,) names; zeros for a sequence without tokens.  With a window over the last
        `window` of them and the first `sinks` only, as `attention` takes it (no weights, and `out` is memory of its own).

        weights (B, H_kv, L) float32, tokens contiguous: every token's softmax weight, summed over the query heads of its KV
        head, is added in place (tokens from L on have no place in it); meanwhile the step keeps 4 bytes for each of L places and query heads, so
        that weights of a large capacity are best given as weights[..., :longest].  max_len bounds the lengths for the plan of the
        splits: without it the width of the table does.  out: memory of its own, or the query itself.  The `workspace` of a step (`workspace()`) belongs to it alone until
        it has run: graphs that may run at the same time need one each."""
        if window is not None or sinks:
            if weights is not None:
                raise ValueError("weights are summed over whole sequences, not within a window")
            return attend("decode_attention", self, query, None, block_table, seq_lens, scale, window, sinks, n_split, workspace, out, max_len, None)
        fast = _ffi.native()
        if fast is not None and n_split is None and workspace is None and out is None:
            done = fast.exact_decode(query, block_table, seq_lens, self.key_cache, self.value_cache, scale, max_len, weights)
            if done is not None:
                return done
        _ffi.require_gpu(query, "query")
        if query.dim() != 3:
            raise ValueError("query must be (B, Hq, d)")
        B, Hq, d = query.shape
        if d != self.head_dim or Hq == 0 or Hq % self.num_kv_heads:
            raise ValueError(f"Incompatible GQA shapes: Q={Hq}, H_kv={self.num_kv_heads}, d={d}")
        if query.dtype != self.dtype or query.device != self.device:
            raise TypeError("the query must have the cache's dtype and live on its GPU")
        _ffi.require_constant("decode_attention", query=query, weights=weights, out=out, key_cache=self.key_cache, value_cache=self.value_cache)
        table, bt_stride, lens = self._sequences(block_table, seq_lens, B)
        if scale is None:
            scale = 1.0 / math.sqrt(d)
        query = query.contiguous().resolve_neg()
        if query.data_ptr() % 16:
            query = query.clone()
        if out is None:
            out = torch.empty_like(query)
        elif (out.shape != query.shape or out.dtype != query.dtype or out.device != query.device or not out.is_contiguous() or
              out.data_ptr() % 16):
            raise ValueError("out must be like the query: contiguous, same shape, dtype and GPU")
        elif out.is_neg():
            raise ValueError("out is negated lazily: its memory does not hold its values")
        else:
            first, end = memory_of(out)
            for name, t in (("query", query), ("weights", weights), ("key_cache", self.key_cache), ("value_cache", self.value_cache), ("block_table", table),
                            ("seq_lens", lens)):
                if t is None or t.numel() == 0 or out.numel() == 0 or (t is query and t.data_ptr() == first):
                    continue                                     # (over the query itself: a row is read by those that write it, and before)
                a, b = memory_of(t)
                if first < b and a < end:
                    raise ValueError(f"out must be memory of its own or the query itself, it overlaps {name}")
        w_ptr, w_b, w_h, w_len = None, 0, 0, 0
        if weights is not None:
            self._weights(weights, B)
            w_ptr, (w_b, w_h), w_len = weights.data_ptr(), weights.stride()[:2], min(weights.shape[2], table.shape[-1] * PAGE_TOKENS)
        if max_len is None:
            max_len = table.shape[-1] * PAGE_TOKENS
        if B == 0:
            return out
        splits = 0 if n_split is None else int(n_split)
        need = self._decode_bytes(B, Hq, max_len, splits, w_len)
        if workspace is None:
            workspace = torch.empty(need // 4, dtype=torch.float32, device=self.device)
        else:
            check_workspace(workspace, need, self.device)
            for name, t in dict(query=query, out=out, weights=weights, block_table=table, seq_lens=lens, **self.tensors()).items():
                if t is not None and overlaps(workspace, t):
                    raise ValueError(f"the workspace overlaps {name}")
        with _ffi.on_device(self.device):
            _ffi.check(_ffi.lib().tq_exact_decode(
                query.data_ptr(), self._tag, B, Hq, self.num_kv_heads, d, self.key_cache.data_ptr(), self.value_cache.data_ptr(),
                *self._strides[:3], self.num_blocks, table.data_ptr(), bt_stride, lens.data_ptr(), float(scale), int(max_len),
                w_ptr, w_b, w_h, w_len, out.data_ptr(), workspace.data_ptr(), splits, _ffi.stream_ptr(self.device)),
                "tq_exact_decode")
        _ffi.changed(out)
        if weights is not None:
            _ffi.changed(weights)
        return out

    def _decode_bytes(self, B, Hq, max_len, splits, weight_len) -> int:
        if splits < 0 or max_len < 0:
            raise ValueError(f"n_split and max_len must not be negative, got {splits} and {max_len}")
        need = _ffi.lib().tq_exact_decode_bytes(self._tag, B, Hq, self.num_kv_heads, self.head_dim, int(max_len), splits, weight_len)
        if need == 0:
            raise ValueError(f"no plan for {B} x {Hq} query heads, max_len {max_len}, n_split {splits}")
        return need

    def attention(self, query: torch.Tensor, query_start_loc: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                  scale: Optional[float] = None, window: Optional[int] = None, sinks: int = 0, n_split: Optional[int] = None,
                  workspace: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, max_len: Optional[int] = None,
                  max_rows: Optional[int] = None) -> torch.Tensor:
        """softmax(scale * q K^T) V for the rows of a step, query (rows, Hq, d) in the cache's dtype (fp16 or bf16; head_dim 64, 128, 192 or 256), whose keys and
        values are in the blocks: row i of sequence b's n = query_start_loc[b + 1] - query_start_loc[b] stands at position p = seq_lens[b] - n + i and sees the
        tokens up to its own; with a window only those behind p - window, and the first `sinks`.  A row that sees nothing is zeros.  Rows
        behind the last sequence are zeros, or left as they are in a given `out`, which is memory of its own.

        max_len and max_rows bound the lengths and a sequence's rows for the plan of the splits (without them the table's width and all rows
        do).  Of up to 32 rows x heads on a KV head and in decode steps the softmax's weights go into the product with the values as two numbers of the cache's
        type, otherwise as one, half a step off.  The `workspace` of a step (`step_workspace()` of the same sizes and bounds) belongs to it alone until it has run: graphs that may
        run at the same time need one each."""
        return attend("attention", self, query, query_start_loc, block_table, seq_lens, scale, window, sinks, n_split, workspace, out, max_len, max_rows)

    def step_workspace(self, rows: int, Hq: int, max_len: int, B: Optional[int] = None, max_rows: Optional[int] = None, window: Optional[int] = None,
                       sinks: int = 0, n_split: Optional[int] = None) -> torch.Tensor:
        """A workspace for `attention` of this size over B sequences, or, without B, for `decode_attention` within a window."""
        window, sinks = seen_by(window, sinks)
        need = plan_bytes(self, self.dtype, B is not None, rows, rows if B is None else B, Hq, max_len, rows if max_rows is None else max_rows, window, sinks,
                          n_split or 0)
        return torch.empty(need // 4, dtype=torch.float32, device=self.device)

    def tensors(self) -> dict:
        return dict(key_cache=self.key_cache, value_cache=self.value_cache)

    def operands(self):
        return self.key_cache, self.value_cache, None, None

    def _memory(self):
        return self.key_cache.data_ptr(), self.value_cache.data_ptr(), None, None

    def workspace(self, B: int, Hq: int, max_len: int, n_split: Optional[int] = None, weight_len: int = 0) -> torch.Tensor:
        """A workspace for decode steps of this size; weight_len: the last dimension of `weights`, 0 without them."""
        return torch.empty(self._decode_bytes(B, Hq, max_len, n_split or 0, weight_len) // 4, dtype=torch.float32, device=self.device)

    def add_window_weights(self, query: torch.Tensor, query_start_loc: torch.Tensor, block_table: torch.Tensor,
                           seq_lens: torch.Tensor, weights: torch.Tensor, window: int, scale: Optional[float] = None,
                           max_len: Optional[int] = None) -> torch.Tensor:
        """Add to `weights` (as in decode_attention) the softmax weight that the newest `window` queries of every sequence
        give to its tokens, summed over those queries and the query heads of a KV head: what there is to evict by
        before the first token is decoded.  query (rows, Hq, d) holds the rows of an engine's step, sequence b's from
        query_start_loc[b] to query_start_loc[b + 1], the last of them at position seq_lens[b] - 1; a query sees the tokens up
        to its own.  A sequence with fewer rows gives those, one without rows nothing."""
        fast = _ffi.native()
        if fast is not None and fast.exact_window(query, query_start_loc, block_table, seq_lens, self.key_cache, self.value_cache, weights,
                                                  window, scale, max_len):
            return weights
        _ffi.require_gpu(query, "query")
        if query.dim() != 3:
            raise ValueError("query must be (rows, Hq, d)")
        rows, Hq, d = query.shape
        if d != self.head_dim or Hq == 0 or Hq % self.num_kv_heads:
            raise ValueError(f"Incompatible GQA shapes: Q={Hq}, H_kv={self.num_kv_heads}, d={d}")
        if query.dtype != self.dtype or query.device != self.device:
            raise TypeError("the query must have the cache's dtype and live on its GPU")
        _ffi.require_constant("add_window_weights", query=query, weights=weights, key_cache=self.key_cache)
        if query_start_loc.dim() != 1 or query_start_loc.shape[0] < 1:
            raise ValueError("query_start_loc must have one entry more than there are sequences")
        B = query_start_loc.shape[0] - 1
        table, bt_stride, lens = self._sequences(block_table, seq_lens, B)
        self._weights(weights, B)
        if not 1 <= window <= MAX_WINDOW:
            raise ValueError(f"window must be 1 .. {MAX_WINDOW}, got {window}")
        if scale is None:
            scale = 1.0 / math.sqrt(d)
        if max_len is None:
            max_len = table.shape[-1] * PAGE_TOKENS
        if B == 0 or rows == 0:
            return weights
        query = query.contiguous().resolve_neg()
        if query.data_ptr() % 16:
            query = query.clone()
        starts = query_start_loc.to(device=self.device, dtype=torch.int32).contiguous().resolve_neg()
        need = _ffi.lib().tq_exact_window_bytes(self._tag, B, Hq, self.num_kv_heads, d, int(window), int(max_len)) if max_len >= 0 else 0
        if need == 0:
            raise ValueError(f"no plan for {B} sequences of {Hq} query heads, window {window}, max_len {max_len}")
        workspace = torch.empty(need // 4, dtype=torch.float32, device=self.device)
        with _ffi.on_device(self.device):
            _ffi.check(_ffi.lib().tq_exact_window(
                query.data_ptr(), self._tag, rows, starts.data_ptr(), B, Hq, self.num_kv_heads, d, int(window), self.key_cache.data_ptr(),
                *self._strides[:3], self.num_blocks, table.data_ptr(), bt_stride, lens.data_ptr(), float(scale), int(max_len),
                weights.data_ptr(), weights.stride(0), weights.stride(1), weights.shape[2], workspace.data_ptr(),
                _ffi.stream_ptr(self.device)), "tq_exact_window")
        _ffi.changed(weights)
        return weights

    # ---- eviction --------------------------------------------------------------------------------------------------------
    def move_tokens(self, evictions: Evictions, block_table: torch.Tensor) -> None:
        """Carry out the moves of `select_evictions` in these blocks, in place.  The sequences' blocks must be their own: a
        block that two sequences share would change for both."""
        fast = _ffi.native()
        if fast is not None and fast.move_exact(self.key_cache, self.value_cache, block_table, evictions.count, evictions.dst, evictions.src):
            return
        _ffi.require_constant("move_tokens", key_cache=self.key_cache, value_cache=self.value_cache)
        count, dst, src, table, bt_stride = evictions.for_cache(block_table, self.num_kv_heads, self.device)
        B, H, moves = dst.shape
        if B == 0:
            return
        with _ffi.on_device(self.device):
            _ffi.check(_ffi.lib().tq_move_tokens_exact(
                self.key_cache.data_ptr(), self.value_cache.data_ptr(), self._tag, self.head_dim, *self._strides[:3], self.num_blocks,
                table.data_ptr(), bt_stride, count.data_ptr(), dst.data_ptr(), src.data_ptr(), B, H, moves, _ffi.stream_ptr(self.device)),
                "tq_move_tokens_exact")
        _ffi.changed(self.key_cache, self.value_cache)
