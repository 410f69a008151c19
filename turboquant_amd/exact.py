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
        if block_table.dtype != torch.int32 or block_table.dim() not in (1, 2) or block_table.shape[-1] == 0:
            raise ValueError("block_table must be int32 (B, max_pages), or (max_pages,) for all sequences")
        if block_table.dim() == 2 and block_table.shape[0] != batch:
            raise ValueError(f"block_table has {block_table.shape[0]} rows for {batch} sequences")
        if seq_lens.shape != (batch,):
            raise ValueError(f"seq_lens must have one entry for each of {batch} sequences")
        _ffi.require_gpu(block_table, "block_table")
        if block_table.device != self.device:
            raise ValueError(f"block_table lives on {block_table.device}, the cache on {self.device}")
        table = block_table.contiguous().resolve_neg()
        lens = seq_lens.to(device=self.device, dtype=torch.int32).contiguous().resolve_neg()
        return table, (-table.shape[0] if table.dim() == 1 else table.shape[1]), lens

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
                         out: Optional[torch.Tensor] = None, max_len: Optional[int] = None) -> torch.Tensor:
        """softmax(scale * q K^T) V for one query token per sequence, query (B, Hq, d) in the cache's dtype, over the
        seq_lens[b] tokens that block_table (B, max_pages) or (max_pages,) names; zeros for a sequence without tokens.

        weights (B, H_kv, L) float32, tokens contiguous: every token's softmax weight, summed over the query heads of its KV
        head, is added in place (tokens from L on have no place in it); meanwhile the step keeps 4 bytes for each of L places and query heads, so
        that weights of a large capacity are best given as weights[..., :longest].  max_len bounds the lengths for the plan of the
        splits: without it the width of the table does.  out: memory of its own, or the query itself.  The `workspace` of a step (`workspace()`) belongs to it alone until
        it has run: graphs that may run at the same time need one each."""
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
            for name, t in (("query", query), ("weights", weights), ("key_cache", self.key_cache), ("value_cache", self.value_cache)):
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
            self._check_workspace(workspace, need)
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

    def _check_workspace(self, workspace: torch.Tensor, need: int) -> None:
        _ffi.require_gpu(workspace, "workspace")
        have = workspace.numel() * workspace.element_size()
        if have < need:
            raise ValueError(f"the workspace holds {have} bytes, this step takes {need}")
        if workspace.device != self.device or not workspace.is_contiguous() or workspace.data_ptr() % 16:
            raise ValueError("the workspace must be contiguous, on a 16-byte boundary and on the cache's GPU")
