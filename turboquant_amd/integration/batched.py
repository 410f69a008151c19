"""Batch-aware attention hooks over the paged compressed pool (new design).

The reference's hooks keep ONE sequence per layer: one store and one ring, and
"prefill vs decode" is `num_tokens > 1` (integration/vllm.py:130-145); that is
what `turboquant_amd.integration.vllm` mirrors.  A serving engine decodes many
sequences per step through block tables.  This module is the batch-aware
counterpart on the same duck-typed contract (integration/vllm.py:361-441):
every hooked standard-attention layer owns a `PagedKVPool` whose page numbers
ARE the engine's block numbers (block size 16 = page size), written from the
K/V tensors of every step and read by the fused decode kernel with the engine's
own block table and sequence lengths.

Besides `num_actual_tokens` and `max_query_len`, `attn_metadata` must carry

  seq_lens        (B,)   int32  length of each sequence INCLUDING this step's tokens
  block_table     (B, max_blocks) int32
  query_start_loc (B+1,) int32  row range of each sequence in the step's token-major tensors

(optionally `seq_lens_cpu` / `query_start_loc_cpu`, which spare a device read on
prefill steps).  Modes are those of `integration.vllm`:

  off           nothing is written, the backend answers
  capture_only  pages are written, the backend answers
  hybrid        decode steps are answered from the pool, the last `ring_capacity`
                tokens of each sequence exactly from the engine's paged cache
                (layout (2, num_blocks, 16, H_kv, d)); prefill by the backend
  full_tq       decode steps are answered from the pool alone; prefill by the
                backend, or by dense causal attention over the step's own K/V
                when the engine's cache was never allocated (`no_alloc`)

The first `exact_layers` layers may stay uncompressed: their decode steps are answered from the engine's paged cache, all of it exactly
(`ExactPagedCache`).  The next `fp8_layers` may keep 8 bits instead of two to four (`Fp8PagedCache`): their decode steps are answered from
those in both modes, and with `no_alloc` their prompts, too, later chunks included.  Both honour the sliding window that a layer's backend names.  And a cache may be cut: `track_weights` has every layer sum the attention weight that its tokens get - from the newest
`window` queries of a prompt's chunk in every step, and in exact layers from every decoded token, whoever else is in the step -, and `evict_batched` keeps the sinks, the newest and the heaviest
of a sequence's tokens, in the engine's blocks and in the pages alike.  The engine goes on with the lengths that it returns.
A hybrid step's exact part are a sequence's last `ring_capacity` slots.  Tokens that stay fill the holes of those that go, so that right behind a cut
the newest lie anywhere below the budget and most of them are read from the pages; they are the last slots again once `ring_capacity` more have come.
"""

from __future__ import annotations

import logging
import math
from dataclasses import dataclass
from itertools import accumulate
from typing import Dict, Optional, Tuple

import torch
import torch.nn.functional as F

from .. import _ffi
from ..attend import HEAD_DIMS, seen_by
from ..eviction import begin_rows, check_table, select_evictions
from ..exact import MAX_HEAD_DIM, ExactPagedCache
from ..fp8 import Fp8PagedCache
from ..paged import APPEND, PAGE_TOKENS, PagedKVPool
from ..quantizer import TurboQuantProd
from . import vllm as _single
from .vllm import (MODE_CAPTURE_ONLY, MODE_HYBRID, MODE_OFF, LayerConfig, _bind, _is_mla_impl, _query_heads_of,
                   _unbound)

logger = logging.getLogger("turboquant.integration.batched")


def _host_list(meta, name):
    cpu = getattr(meta, name + "_cpu", None)
    t = cpu if cpu is not None else getattr(meta, name)
    return [int(x) for x in t.tolist()]


def _window_of(name: str, impl) -> Tuple[Optional[int], int]:
    """(window, sinks) of a layer, as its backend names them: `sliding_window`, tokens that a query sees with its own among them, or the pair of
    those on its left and right (-1: all), and `sink_tokens`, first tokens that stay visible."""
    window = getattr(impl, "sliding_window", None)
    if isinstance(window, (tuple, list)):
        left, right = (int(x) for x in window)
        if right > 0:
            raise ValueError(f"{name} sees {right} tokens behind its own: not a causal layer")
        window = left + 1 if left >= 0 else None
    if window is None or int(window) <= 0:
        return None, 0
    window, sinks = int(window), int(getattr(impl, "sink_tokens", 0))
    seen_by(window, sinks)
    return window, sinks


def _names_a_window(impl) -> bool:
    """Whether a layer's backend has its queries see part of the tokens only, in whatever form it says so."""
    window = getattr(impl, "sliding_window", None)
    try:
        if isinstance(window, (tuple, list)):
            return any(int(x) >= 0 for x in window)
        return window is not None and int(window) > 0
    except (TypeError, ValueError, OverflowError):
        return True


@dataclass
class BatchedLayerState:
    """One attention layer: its quantiser and the compressed pool that shadows the engine's blocks, or 8-bit blocks that do (neither: the layer stays exact)."""
    config: LayerConfig
    quantizer: Optional[TurboQuantProd]
    pool: Optional[PagedKVPool]
    tokens_written: int = 0
    decode_steps: int = 0
    weights: Optional[torch.Tensor] = None                     # (B, H_kv, tokens): what every slot's token has been given so far
    positions: Optional[torch.Tensor] = None                   # (B, H_kv, tokens): where in the sequence it stood
    window: int = 0
    blocks_current: bool = True                                # the engine's blocks hold a step's tokens before its attention: do_kv_cache_update
    fp8: Optional[Fp8PagedCache] = None
    sees: Tuple[Optional[int], int] = (None, 0)                # sliding window and sinks of an exact or 8-bit layer

    @property
    def supports_hybrid(self) -> bool:
        """Whether the engine's cache may be freed (an exact layer has nothing else)."""
        return self.pool is not None or self.fp8 is not None

    # ---- write -------------------------------------------------------------------
    def write(self, key: torch.Tensor, value: torch.Tensor, meta) -> None:
        """Quantise this step's tokens (n, H_kv, d) into the pages their sequences own."""
        cfg = self.config
        n = int(meta.num_actual_tokens)
        self.check_step(meta)
        if self.pool is None and self.fp8 is None:             # the engine's own cache has them
            self.tokens_written += n
            return
        k = key[:n].reshape(n, cfg.num_kv_heads, cfg.head_dim)
        v = value[:n].reshape(n, cfg.num_kv_heads, cfg.head_dim)
        table = meta.block_table
        if self.fp8 is not None:
            self.fp8.write(k, v, meta.query_start_loc, table, meta.seq_lens)
        elif int(meta.max_query_len) == 1:                       # one token per sequence: a single batched append
            k, v, lens = k[:, None], v[:, None], meta.seq_lens
            if not (_ffi.as_defined(self.pool, APPEND) and self.pool._append_newest(k, v, table, lens)):
                self.pool.append(k, v, table, start_pos=lens.to(torch.int32) - 1)
        else:                                                  # ragged rows: still one call, nothing read back
            qsl = meta.query_start_loc.to(device=k.device, dtype=torch.int32)
            run = qsl[1:] - qsl[:-1]
            start = meta.seq_lens.to(device=k.device, dtype=torch.int32) - run
            self.pool.append_ragged(k, v, qsl[:-1], run, start, table, max_run=int(meta.max_query_len))
        self.tokens_written += n

    def ingest_paged_cache(self, kv_cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                           max_tokens: Optional[int] = None) -> None:
        """Compress what the engine's exact paged cache (2, num_blocks, 16, H_kv, d) already holds for the
        sequences of `block_table`: tokens [0, seq_lens[b]) of every sequence, read in place through the
        block table and written to the pages of the same numbers (the batch counterpart of
        capture.py:187-217, without the gather copy; 8-bit layers gather pieces of them).  max_tokens: the first tokens of every sequence only."""
        if not self.supports_hybrid:
            raise RuntimeError("an exact layer has no pages to write to")
        if self.fp8 is not None:
            most = math.inf if max_tokens is None else max_tokens
            self._ingest_fp8(kv_cache, block_table, [min(int(n), most) for n in seq_lens.tolist()])
            return
        self.pool.append_from_blocks(kv_cache[0], kv_cache[1], block_table, block_table, seq_lens,
                                     max_tokens=max_tokens)
        self.tokens_written += int(seq_lens.sum())

    def _ingest_fp8(self, kv_cache, block_table, lens) -> None:
        """All sequences together, whole blocks of each (none is rounded twice) up to 65536 rows in all, gathered from their blocks."""
        B, device = len(lens), self.fp8.device
        if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.shape[0] < B or block_table.shape[1] == 0 or block_table.device != device:
            raise ValueError(f"block_table must be int32 ({B}, max_pages) on {device}")
        table, num_blocks = block_table[:B], kv_cache.shape[1]
        piece = max(1, 65536 // PAGE_TOKENS // max(1, B)) * PAGE_TOKENS
        for first in range(0, max(lens, default=0), piece):
            runs = [max(0, min(n - first, piece)) for n in lens]
            step = torch.tensor([0, *accumulate(runs), *(first + n for n in runs)], dtype=torch.int32).to(device)
            starts, row = step[: B + 1], torch.arange(sum(runs), dtype=torch.int32, device=device)
            b = torch.searchsorted(starts[1:].contiguous(), row, right=True)
            t = (first + row - starts[b]).long()
            # (tokens without a block read one that is there, and are not written)
            block = table[b, (t // PAGE_TOKENS).clamp_max(table.shape[1] - 1)].long().clamp(0, num_blocks - 1)
            self.fp8.write(kv_cache[0][block, t % PAGE_TOKENS], kv_cache[1][block, t % PAGE_TOKENS], starts, table, step[B + 1:])
            self.tokens_written += sum(runs)

    # ---- read --------------------------------------------------------------------
    def _exact_tail(self, kv_cache, meta):
        """The last `ring_capacity` tokens of every sequence from the engine's paged cache:
        (B, R, H_kv, d) keys and values, their valid counts, and the compressed lengths."""
        cfg = self.config
        R = cfg.ring_capacity
        ok = (torch.is_tensor(kv_cache) and kv_cache.dim() == 5 and kv_cache.shape[0] == 2 and
              kv_cache.shape[2] == PAGE_TOKENS and kv_cache.shape[3] == cfg.num_kv_heads and
              kv_cache.shape[4] == cfg.head_dim)
        if not ok or R <= 0:
            return None
        seq = meta.seq_lens.to(torch.int64)
        tail = torch.clamp(seq, max=R)                                          # (B,)
        pos = (seq - tail)[:, None] + torch.arange(R, device=seq.device)[None]  # (B, R) token positions
        pos = torch.minimum(pos, (seq - 1).clamp_min(0)[:, None])
        blocks = torch.gather(meta.block_table.to(torch.int64), 1, pos // PAGE_TOKENS)
        slot = blocks * PAGE_TOKENS + pos % PAGE_TOKENS
        flat_k = kv_cache[0].reshape(-1, cfg.num_kv_heads, cfg.head_dim)
        flat_v = kv_cache[1].reshape(-1, cfg.num_kv_heads, cfg.head_dim)
        return flat_k[slot], flat_v[slot], tail.to(torch.int32), (seq - tail).to(torch.int32)

    def attend(self, query: torch.Tensor, meta, scale: Optional[float] = None, kv_cache=None,
               hybrid: bool = False) -> torch.Tensor:
        """One query token per sequence, (B, H_q, d) -> (B, H_q, d)."""
        self.decode_steps += 1
        cfg = self.config
        window, sinks = self.sees
        if self.fp8 is not None:
            return self.fp8.decode_attention(query, meta.block_table, meta.seq_lens, scale=scale, window=window, sinks=sinks,
                                             max_len=getattr(meta, "max_seq_len", None))
        if self.pool is None:
            longest, weights = getattr(meta, "max_seq_len", None), self.weights
            if window is not None:
                return ExactPagedCache.from_engine(kv_cache).decode_attention(query, meta.block_table, meta.seq_lens, scale=scale, window=window, sinks=sinks,
                                                                              max_len=longest)
            if weights is not None:                            # (the step keeps a score for every place; check_step has seen that there are no longer sequences)
                weights = weights[: query.shape[0], :, : max(1, longest) if longest is not None else None]
            return ExactPagedCache.from_engine(kv_cache).decode_attention(query, meta.block_table, meta.seq_lens, scale=scale, weights=weights, max_len=longest)
        if (hybrid and cfg.ring_capacity > 0 and torch.is_tensor(kv_cache) and kv_cache.dim() == 5 and
                kv_cache.shape[0] == 2 and tuple(kv_cache.shape[2:]) == (PAGE_TOKENS, cfg.num_kv_heads, cfg.head_dim) and
                kv_cache.dtype == query.dtype and cfg.ring_capacity <= 1024 and
                self.pool.ring_cache_ok(kv_cache[0], kv_cache[1])):
            # the exact tokens are read in place from the engine's cache, through the step's block table
            return self.pool.decode_attention_ring(query, meta.block_table, meta.seq_lens, kv_cache[0], kv_cache[1],
                                                   cfg.ring_capacity, scale=scale,
                                                   max_len=getattr(meta, "max_seq_len", None))
        recent = self._exact_tail(kv_cache, meta) if hybrid else None
        if recent is None:
            return self.pool.decode_attention(query, meta.block_table, meta.seq_lens, scale=scale,
                                              max_len=getattr(meta, "max_seq_len", None))
        rk, rv, rlen, hist = recent
        return self.pool.decode_attention(query, meta.block_table, hist, scale=scale, recent_k=rk, recent_v=rv,
                                          recent_len=rlen, max_len=getattr(meta, "max_seq_len", None))

    def attend_rows(self, query: torch.Tensor, meta, scale: Optional[float] = None) -> torch.Tensor:
        """The rows of a step, (n, H_q, d) -> (n, H_q, d), from the 8-bit blocks alone: prompts, chunks of them, single tokens beside them."""
        window, sinks = self.sees
        return self.fp8.attention(query, meta.query_start_loc, meta.block_table, meta.seq_lens, scale=scale, window=window, sinks=sinks,
                                  max_len=getattr(meta, "max_seq_len", None), max_rows=int(meta.max_query_len))

    # ---- eviction ------------------------------------------------------------------
    def track(self, batch: int, max_len: int, window: int) -> None:
        """Sum weights from now on, for up to `batch` sequences (rows of the step's block table) of up to max_len tokens."""
        shape = (batch, self.config.num_kv_heads, max_len)
        self.weights = torch.zeros(shape, dtype=torch.float32, device=self.config.device)
        self.positions = torch.arange(max_len, dtype=torch.int32, device=self.config.device).expand(shape).contiguous()
        self.window = window

    def check_step(self, meta) -> None:
        """Whether what is tracked has room for this step."""
        if self.weights is None:
            return
        rows = meta.seq_lens.shape[0]
        if rows > self.weights.shape[0]:
            raise ValueError(f"a step of {rows} rows where {self.weights.shape[0]} are tracked")
        longest = getattr(meta, "max_seq_len", None)
        if longest is None:                                    # (what the lengths may be, without waiting for the GPU)
            lens = getattr(meta, "seq_lens_cpu", None)
            longest = meta.block_table.shape[-1] * PAGE_TOKENS if lens is None else max((int(n) for n in lens), default=0)
        self.check_length(int(longest))

    def check_length(self, longest: int) -> None:
        if longest > self.weights.shape[2]:
            raise ValueError(f"a sequence of up to {longest} tokens where {self.weights.shape[2]} are tracked: the newest would have no weight and no position")

    def begin(self, meta) -> None:
        """Rows whose sequence begins in this step have had nothing."""
        rows = meta.seq_lens.shape[0]
        begin_rows(self.weights[:rows], self.positions[:rows], meta.seq_lens, meta.query_start_loc)

    def reorder(self, order: torch.Tensor) -> None:
        """Row i goes on with what row order[i] has had; -1: with nothing."""
        none = order < 0
        at = order.clamp_min(0)
        fresh = torch.arange(self.positions.shape[2], dtype=torch.int32, device=self.positions.device)
        self.weights.copy_(self.weights[at].masked_fill_(none[:, None, None], 0))
        self.positions.copy_(torch.where(none[:, None, None], fresh, self.positions[at]))

    def observe(self, query: torch.Tensor, meta, kv_cache: torch.Tensor, scale: Optional[float] = None) -> None:
        """Add the weights that the newest queries of every sequence in this step give; query (rows, H_q, d).  Compressed layers: of every sequence with
        more than one row in it."""
        lens, starts = meta.seq_lens, meta.query_start_loc
        if self.pool is not None:
            # One row is a decode step's, which a compressed layer does not count: not beside another sequence's prompt either (a sequence without
            # tokens gives nothing)
            lens, starts = (t.to(self.weights.device) for t in (lens, starts))
            lens = lens.masked_fill(starts[1:] - starts[:-1] == 1, 0)
        ExactPagedCache.from_engine(kv_cache).add_window_weights(query, starts, meta.block_table, lens, self.weights[: lens.shape[0]], window=self.window,
                                                                 scale=scale, max_len=getattr(meta, "max_seq_len", None))

    def prepare_cut(self, block_table: torch.Tensor, seq_lens: torch.Tensor, kv_cache: Optional[torch.Tensor] = None,
                    max_len: Optional[int] = None) -> Optional[ExactPagedCache]:
        """The cache that moves are carried out in, and every check of them: a cut that would fail halfway is not begun."""
        if self.weights is None:
            raise RuntimeError("nothing has been tracked: track_weights comes first")
        rows = block_table.shape[0] if block_table.dim() else 0
        if rows > self.weights.shape[0]:
            raise ValueError(f"a cut of {rows} rows where {self.weights.shape[0]} are tracked")
        check_table(block_table, rows, self.weights.device)
        if max_len is None and not seq_lens.is_cuda:
            max_len = int(seq_lens.max()) if seq_lens.numel() else 0
        if max_len is not None:                                # (lengths on the GPU are those of steps, each of which was checked)
            self.check_length(int(max_len))
        if kv_cache is None:
            if self.pool is None:
                raise ValueError("an exact layer is cut in the engine's cache, (2, num_blocks, 16, H_kv, d): there is none")
            return None
        cache = ExactPagedCache.from_engine(kv_cache)
        if cache.num_kv_heads != self.config.num_kv_heads or cache.device != self.weights.device:
            raise ValueError(f"a cache of {cache.num_kv_heads} KV heads on {cache.device} for a layer of {self.config.num_kv_heads} on {self.weights.device}")
        return cache

    def evict(self, block_table: torch.Tensor, seq_lens: torch.Tensor, budget: int, seen: Optional[torch.Tensor] = None, sinks: int = 4,
              recent: int = 0, kv_cache: Optional[torch.Tensor] = None, max_len: Optional[int] = None) -> torch.Tensor:
        """Cut every sequence to `budget` tokens (`select_evictions`), in the engine's cache (2, num_blocks, 16, H_kv, d), if there is one (an exact layer
        has nothing else), and in this layer's pages; returns the lengths that are left.  max_len: a bound on seq_lens, checked against what is
        tracked without waiting for the GPU."""
        return self.cut(self.prepare_cut(block_table, seq_lens, kv_cache, max_len), block_table, seq_lens, budget, seen, sinks, recent)

    def cut(self, cache: Optional[ExactPagedCache], block_table, seq_lens, budget, seen, sinks, recent) -> torch.Tensor:
        """`evict` behind its `prepare_cut`."""
        held = self.weights[: block_table.shape[0]], self.positions[: block_table.shape[0]]
        e = select_evictions(*held, seq_lens, budget, seen=seen, sinks=sinks, recent=recent, out=held)
        if cache is not None:
            cache.move_tokens(e, block_table)
        if self.pool is not None:
            self.pool.move_tokens(e, block_table)
        return e.lens

    def memory_bytes(self) -> int:
        if self.fp8 is not None:
            return self.fp8.memory_bytes()
        return 0 if self.pool is None else self.pool.data.numel()


class _BatchedLayerHooks:
    """Replacement methods of one standard attention layer (impl first, like the unbound originals)."""

    def __init__(self, state: BatchedLayerState, orig_forward, orig_update, no_alloc: bool):
        self.state, self.orig_forward, self.orig_update, self.no_alloc = state, orig_forward, orig_update, no_alloc

    def kv_update(self, impl, layer, key, value, kv_cache, slot_mapping):
        if not self.no_alloc:                                  # the engine's exact cache stays current
            self.orig_update(impl, layer, key, value, kv_cache, slot_mapping)

    def _deliver(self, result, query, output, n):
        cfg = self.state.config
        flat = result.reshape(n, cfg.num_query_heads * cfg.head_dim).to(query.dtype)
        if output is not None:
            dst = output[:n]
            dst.copy_((result if dst.dim() == 3 else flat).to(dst.dtype))
            return output
        return result.to(query.dtype) if query.dim() == 3 else flat

    def _dense_prefill(self, impl, query, key, value, meta, n):
        """Causal attention of every sequence over its own rows of this step (first chunk of a
        sequence only: there is no exact cache to read earlier tokens from)."""
        cfg = self.state.config
        q = query[:n].reshape(n, cfg.num_query_heads, cfg.head_dim)
        if self.state.fp8 is not None:                         # (its blocks have the earlier tokens, and this step's are written)
            return self.state.attend_rows(q, meta, getattr(impl, "scale", None))
        k = key[:n].reshape(n, cfg.num_kv_heads, cfg.head_dim)
        v = value[:n].reshape(n, cfg.num_kv_heads, cfg.head_dim)
        rep = cfg.num_query_heads // cfg.num_kv_heads
        scale = getattr(impl, "scale", 1.0 / math.sqrt(cfg.head_dim))
        out = torch.empty_like(q)
        lens, qsl = _host_list(meta, "seq_lens"), _host_list(meta, "query_start_loc")
        for b in range(len(lens)):
            r0, r1 = qsl[b], qsl[b + 1]
            if r1 <= r0:
                continue
            if lens[b] != r1 - r0:
                raise RuntimeError("chunked prefill needs the engine's paged cache (hooks installed with no_alloc)")
            kb, vb = k[r0:r1].repeat_interleave(rep, 1), v[r0:r1].repeat_interleave(rep, 1)
            o = F.scaled_dot_product_attention(q[r0:r1].transpose(0, 1)[None], kb.transpose(0, 1)[None],
                                               vb.transpose(0, 1)[None], is_causal=True, scale=scale)
            out[r0:r1] = o[0].transpose(0, 1)
        return out

    def forward(self, impl, layer, query, key, value, kv_cache, attn_metadata, output=None, output_scale=None,
                output_block_scale=None):
        mode = _single.get_mode()
        passthrough = lambda: self.orig_forward(impl, layer, query, key, value, kv_cache, attn_metadata, output,
                                                output_scale, output_block_scale)
        if mode == MODE_OFF or attn_metadata is None:          # None = the engine's profiling pass
            return passthrough()
        self.state.write(key, value, attn_metadata)
        n = int(attn_metadata.num_actual_tokens)
        if self.state.weights is not None:
            self.state.begin(attn_metadata)
            # (an exact layer's decode step adds its weights where it is answered below, unless the backend answers it)
            if int(attn_metadata.max_query_len) > 1 or (self.state.pool is None and mode == MODE_CAPTURE_ONLY):
                cfg = self.state.config
                self.state.observe(query[:n].reshape(n, cfg.num_query_heads, cfg.head_dim), attn_metadata, kv_cache, getattr(impl, "scale", None))
        if mode == MODE_CAPTURE_ONLY:
            return passthrough()
        if int(attn_metadata.max_query_len) > 1:               # prefill (or a mixed step): exact attention
            if not self.no_alloc:
                return passthrough()
            return self._deliver(self._dense_prefill(impl, query, key, value, attn_metadata, n), query, output, n)
        cfg = self.state.config
        q = query[:n].reshape(n, cfg.num_query_heads, cfg.head_dim)
        result = self.state.attend(q, attn_metadata, scale=getattr(impl, "scale", None), kv_cache=kv_cache,
                                   hybrid=(mode == MODE_HYBRID and not self.no_alloc))
        return self._deliver(result, query, output, n)


def install_batched_hooks(model_runner, num_blocks: int, key_bits: int = 3, value_bits: int = 2,
                          value_group_size: int = 32, ring_capacity: int = 128, initial_layers_count: int = 4,
                          initial_layers_key_bits: Optional[int] = None, mode: str = MODE_CAPTURE_ONLY,
                          no_alloc: bool = False, dtype: torch.dtype = torch.bfloat16,
                          exact_layers: int = 0, fp8_layers: int = 0) -> Dict[str, BatchedLayerState]:
    """Hook every standard attention layer of `model_runner` with a compressed pool of `num_blocks`
    16-token pages (the engine's block count); returns {layer name: BatchedLayerState}.  Bit widths are
    assigned as by `install_hooks` (integration/vllm.py:333-359).  The first `exact_layers` of them get no pool: their
    decode steps are answered from the engine's cache.  The next `fp8_layers` keep e4m3 blocks of the engine's numbers instead of pages, and have head sizes of
    64, 128, 192 or 256.  Latent-attention layers are left alone.  A layer can stay exact
    only if its backend has do_kv_cache_update and its head size is a multiple of 64 up to 768.

    A backend's `sliding_window` (and `sink_tokens`) hold for exact and 8-bit layers (at those four head sizes); pages of two to four bits
    are attended to as a whole, which a warning says of layers whose backend names a window: their decode steps see more tokens in `hybrid` and `full_tq` than the backend's."""
    if exact_layers < 0 or fp8_layers < 0:
        raise ValueError(f"exact_layers and fp8_layers must not be negative, got {exact_layers} and {fp8_layers}")
    if exact_layers and no_alloc:
        raise ValueError("exact layers are answered from the engine's cache, which no_alloc leaves out")
    if fp8_layers and torch.device(model_runner.device).type != "cuda":
        raise ValueError(f"8-bit layers need a GPU, the model runs on {model_runner.device}")
    layers, whole = [], []
    for name, module in model_runner.compilation_config.static_forward_context.items():
        impl = getattr(module, "impl", None)
        if impl is None or getattr(impl, "num_kv_heads", None) is None or not hasattr(impl, "head_size"):
            continue
        if _is_mla_impl(impl):
            continue
        if len(layers) < exact_layers and not hasattr(impl, "do_kv_cache_update"):
            raise ValueError(f"{name} cannot stay exact: its backend has no do_kv_cache_update, so that only its forward(), which a decode step does "
                             "not reach, would write the engine's cache")
        if len(layers) < exact_layers and (int(impl.head_size) % 64 or not 0 < int(impl.head_size) <= MAX_HEAD_DIM):
            raise ValueError(f"{name} cannot stay exact: its head_dim {int(impl.head_size)} is no multiple of 64 up to {MAX_HEAD_DIM}")
        idx, sees = len(layers), (None, 0)
        if idx < exact_layers + fp8_layers:
            sees = _window_of(name, impl)
            if int(impl.head_size) not in HEAD_DIMS and (idx >= exact_layers or sees[0] is not None):
                raise ValueError(f"{name}: 8-bit layers and sliding windows take head sizes of {', '.join(map(str, HEAD_DIMS))}, got {int(impl.head_size)}")
        elif _names_a_window(impl):
            whole.append(name)
        layers.append((name, module, impl, sees))
    if whole:
        logger.warning("[TurboQuant] %d layers have a sliding window, which pages of two to four bits do not honour: %s (exact_layers and fp8_layers do)", len(whole),
                       ", ".join(whole))
    _single.set_mode(mode)
    if initial_layers_key_bits is None:
        initial_layers_key_bits = min(key_bits + 1, 4)
    states: Dict[str, BatchedLayerState] = {}
    device = torch.device(model_runner.device)
    for idx, (name, module, impl, sees) in enumerate(layers):
        head_dim = int(impl.head_size)
        cfg = LayerConfig(head_dim=head_dim, num_kv_heads=int(impl.num_kv_heads),
                          num_query_heads=_query_heads_of(module, impl),
                          key_bits=initial_layers_key_bits if idx < initial_layers_count else key_bits,
                          value_bits=value_bits, value_group_size=min(value_group_size, head_dim),
                          ring_capacity=ring_capacity, layer_idx=idx, backend_kind="flash", device=device)
        tq = pool = fp8 = None
        if exact_layers <= idx < exact_layers + fp8_layers:
            fp8 = Fp8PagedCache.allocate(num_blocks, cfg.num_kv_heads, head_dim, device)
        elif idx >= exact_layers:
            tq = TurboQuantProd(head_dim, bits=cfg.key_bits, device=device, seed=42 + 7 * idx)
            pool = PagedKVPool(tq, cfg.num_kv_heads, num_blocks, value_bits=value_bits,
                               value_group_size=cfg.value_group_size, dtype=dtype, device=device)
        has_update = hasattr(impl, "do_kv_cache_update")
        state = BatchedLayerState(config=cfg, quantizer=tq, pool=pool, blocks_current=has_update, fp8=fp8, sees=sees)
        states[name] = state
        hooks = _BatchedLayerHooks(state, _unbound(impl.forward),
                                   _unbound(impl.do_kv_cache_update) if has_update else None, no_alloc)
        if has_update:
            impl.do_kv_cache_update = _bind(impl, hooks.kv_update)
        impl.forward = _bind(impl, hooks.forward)
        impl._tq_layer_state = state
    model_runner._tq_layer_states = states
    model_runner._tq_no_alloc = no_alloc
    logger.info("[TurboQuant] Batched hooks on %d layers (mode=%s, no_alloc=%s)", len(states), mode, no_alloc)
    return states


def track_weights(model_runner, batch: int, max_len: int, window: int = 32) -> None:
    """Have every hooked layer sum the attention weight of its tokens from now on: up to `batch` rows of the block table, up to max_len tokens each
    (a step that may hold longer sequences is refused).  The newest `window` queries of every prompt, or of its chunk in a step, add what they give, read
    from the engine's cache; a decoding sequence's query adds its own in exact layers, in compressed ones not: their generated tokens have only the
    weight that later prompt chunks give them, so `recent` is what keeps them.

    What is summed belongs to a row.  A row whose sequence begins in a step (all of its tokens are that step's) starts anew; an engine that
    gives rows of sequences that go on to others - a batch closed up, two rows swapped, a sequence that begins behind tokens it did not compute - says so
    with `reorder_rows` before the next step."""
    if getattr(model_runner, "_tq_no_alloc", False):
        raise ValueError("weights are summed over the engine's cache, which no_alloc leaves out")
    if not 1 <= window <= 1024:
        raise ValueError(f"window must be 1 .. 1024, got {window}")
    for name, state in model_runner._tq_layer_states.items():
        if state.fp8 is not None:
            raise ValueError(f"8-bit layers cannot be cut: the tokens of {name} would not move with the others")
        if state.sees[0] is not None:
            raise ValueError(f"layers with a sliding window cannot be cut: {name} tells by a token's slot how far behind it is")
        if not state.blocks_current:
            raise ValueError(f"weights are summed over the engine's cache before a step's attention: {name}, whose backend has no do_kv_cache_update, "
                             "writes it too late")
    for state in model_runner._tq_layer_states.values():
        state.track(batch, max_len, window)


def reorder_rows(model_runner, order) -> None:
    """The rows of the batch have changed places: row i is now what row order[i] was, or, with -1, a sequence of which nothing has been summed.  order has
    an entry for each tracked row, none of them twice."""
    states = list(model_runner._tq_layer_states.values())
    if not states or any(s.weights is None for s in states):
        raise RuntimeError("nothing has been tracked: track_weights comes first")
    order = [int(i) for i in order]
    rows, taken = states[0].weights.shape[0], [i for i in order if i >= 0]
    if len(order) != rows or any(not -1 <= i < rows for i in order) or len(set(taken)) != len(taken):
        raise ValueError(f"order must name each of {rows} rows once at most, or -1, got {order}")
    for s in states:
        s.reorder(torch.tensor(order, device=s.weights.device))


def evict_batched(model_runner, block_table: torch.Tensor, seq_lens: torch.Tensor, budget: int, seen: Optional[torch.Tensor] = None,
                  sinks: int = 4, recent: int = 0, max_len: Optional[int] = None) -> torch.Tensor:
    """Cut every sequence to `budget` tokens in every hooked layer, each KV head by its own weights; returns the lengths (B,) that all layers have
    now.  seq_lens (B,) tokens held, seen (B,) tokens had in all (None: nothing was cut before).  Blocks behind the new lengths are the
    engine's to give away.  A sequence's blocks must be its own (no prefix shared with another).  max_len: a bound on
    seq_lens; one beyond what is tracked is refused (so are lengths on the host, and steps that would lead there)."""
    ctx = model_runner.compilation_config.static_forward_context
    states, caches = model_runner._tq_layer_states, {}
    for name, state in states.items():                         # of all layers, before the first is cut
        held = getattr(ctx[name], "kv_cache", None)
        cache = held if torch.is_tensor(held) else held[0] if held else None
        caches[name] = state.prepare_cut(block_table, seq_lens, cache if torch.is_tensor(cache) and cache.dim() == 5 else None, max_len)
    lens = seq_lens
    for name, state in states.items():
        lens = state.cut(caches[name], block_table, seq_lens, budget, seen, sinks, recent)
    return lens


def get_batched_stats(model_runner) -> dict:
    states = getattr(model_runner, "_tq_layer_states", None) or {}
    return {"num_layers": len(states),
            "tokens_written_per_layer": max((s.tokens_written for s in states.values()), default=0),
            "decode_steps": max((s.decode_steps for s in states.values()), default=0),
            "total_memory_bytes": sum(s.memory_bytes() for s in states.values()),
            "mode": _single.get_mode()}
