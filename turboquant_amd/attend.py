"""What the calls over a paged cache share: a step's sequences, and attention of its rows.

The rows of an engine's step are its sequences' newest tokens: rows query_start_loc[b] .. query_start_loc[b + 1] - 1 are sequence b's, the last of
them token seq_lens[b] - 1.  `ExactPagedCache` (the engine's blocks) and `Fp8PagedCache` (8 bits) answer the same calls.  (New: the reference leaves
prompts, windows and its exact cache to the engine's backend, integration/vllm.py:290-318.)
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from . import _ffi
from .eviction import memory_of
from .paged import PAGE_TOKENS

HEAD_DIMS = (64, 128, 192, 256)
MAX_SCALE = 2.0 ** 127              # (times log2 e it is a number in 32 bits)


def sequences(device: torch.device, block_table: torch.Tensor, seq_lens: torch.Tensor, batch: int):
    """(table, its stride as the library takes it, lengths): int32 on the cache's GPU, contiguous."""
    if block_table.dtype != torch.int32 or block_table.dim() not in (1, 2) or block_table.shape[-1] == 0:
        raise ValueError("block_table must be int32 (B, max_pages), or (max_pages,) for all sequences")
    if block_table.dim() == 2 and block_table.shape[0] != batch:
        raise ValueError(f"block_table has {block_table.shape[0]} rows for {batch} sequences")
    if seq_lens.shape != (batch,):
        raise ValueError(f"seq_lens must have one entry for each of {batch} sequences")
    _ffi.require_gpu(block_table, "block_table")
    if block_table.device != device:
        raise ValueError(f"block_table lives on {block_table.device}, the cache on {device}")
    table = block_table.contiguous().resolve_neg()
    lens = seq_lens.to(device=device, dtype=torch.int32).contiguous().resolve_neg()
    return table, (-table.shape[0] if table.dim() == 1 else table.shape[1]), lens


def step_starts(device: torch.device, query_start_loc: torch.Tensor):
    """(starts, sequences): int32 on the cache's GPU, contiguous."""
    if query_start_loc.dim() != 1 or query_start_loc.shape[0] < 1:
        raise ValueError("query_start_loc must have one entry more than there are sequences")
    if query_start_loc._is_zerotensor():
        raise ValueError("query_start_loc must hold its values")
    return query_start_loc.to(device=device, dtype=torch.int32).contiguous().resolve_neg(), query_start_loc.shape[0] - 1


def check_workspace(workspace: torch.Tensor, need: int, device: torch.device) -> None:
    _ffi.require_gpu(workspace, "workspace")
    have = workspace.numel() * workspace.element_size()
    if have < need:
        raise ValueError(f"the workspace holds {have} bytes, this step takes {need}")
    if workspace.device != device or not workspace.is_contiguous() or workspace.data_ptr() % 16:
        raise ValueError("the workspace must be contiguous, on a 16-byte boundary and on the cache's GPU")


def overlaps(a: torch.Tensor, b: torch.Tensor) -> bool:
    if a.numel() == 0 or b.numel() == 0:
        return False
    x, y = memory_of(a), memory_of(b)
    return x[0] < y[1] and y[0] < x[1]


def row_strides(t: torch.Tensor) -> tuple:
    """Strides of tokens and heads (rows, H, d) as the library takes them: of a dimension of one element torch leaves any number, which nothing goes by."""
    return tuple(s if n > 1 else 0 for s, n in zip(t.stride()[:2], t.shape[:2]))


def seen_by(window: Optional[int], sinks: int):
    """(window as the library takes it, sinks) of a call, checked."""
    if window is None:
        if sinks:
            raise ValueError(f"sinks are what stays visible outside a window: {sinks} without one")
        return 0, 0
    window, sinks = int(window), int(sinks)
    if not 1 <= window < 1 << 31 or not 0 <= sinks < 1 << 31:
        raise ValueError(f"window must be at least 1 and sinks at least 0, both below 2^31, got {window} and {sinks}")
    return window, sinks


def plan_bytes(cache, dtype, starts: bool, rows: int, B: int, Hq: int, max_len: int, max_rows: int, window: int, sinks: int, n_split: int) -> int:
    if n_split < 0 or max_len < 0 or max_rows < 0:
        raise ValueError(f"n_split, max_len and max_rows must not be negative, got {n_split}, {max_len} and {max_rows}")
    need = _ffi.lib().tq_attend_bytes(_ffi.dtype_tag(dtype), cache._tag, int(starts), rows, B, Hq, cache.num_kv_heads, cache.head_dim, int(max_len),
                                      int(max_rows), window, sinks, n_split)
    if need == 0:
        raise ValueError(f"no plan for {rows} rows of {B} sequences, {Hq} query heads on {cache.num_kv_heads}, max_len {max_len}, n_split {n_split}")
    return need


def attend(what: str, cache, query: torch.Tensor, query_start_loc: Optional[torch.Tensor], block_table: torch.Tensor, seq_lens: torch.Tensor,
           scale: Optional[float], window: Optional[int], sinks: int, n_split: Optional[int], workspace: Optional[torch.Tensor],
           out: Optional[torch.Tensor], max_len: Optional[int], max_rows: Optional[int]) -> torch.Tensor:
    """The calls `attention` and `decode_attention` (query_start_loc None) of both caches."""
    fast = _ffi.native()
    if fast is not None and n_split is None and workspace is None and out is None:
        done = fast.attend(query, query_start_loc, block_table, seq_lens, *cache.operands(), scale, window, sinks, max_len, max_rows)
        if done is not None:
            return done
    _ffi.require_gpu(query, "query")
    if query.dim() != 3:
        raise ValueError("query must be (rows, Hq, d)" if query_start_loc is not None else "query must be (B, Hq, d)")
    rows, Hq, d = query.shape
    H, device = cache.num_kv_heads, cache.device
    if d != cache.head_dim or Hq == 0 or Hq % H:
        raise ValueError(f"Incompatible GQA shapes: Q={Hq}, H_kv={H}, d={d}")
    if d not in HEAD_DIMS:
        raise ValueError(f"{what} takes head sizes of {', '.join(map(str, HEAD_DIMS))}, got {d}")
    if query.dtype not in (torch.float16, torch.bfloat16) or cache.dtype not in (query.dtype, torch.float8_e4m3fn):
        raise TypeError(f"{what} takes fp16 or bf16 queries, of the cache's type or over 8 bits, got {query.dtype} over {cache.dtype}")
    if query.device != device:
        raise TypeError("the query must live on the cache's GPU")
    window, sinks = seen_by(window, sinks)
    held = cache.tensors()
    _ffi.require_constant(what, query=query, out=out, **held)
    starts, B = None, rows
    if query_start_loc is not None:
        starts, B = step_starts(device, query_start_loc)
    table, bt_stride, lens = sequences(device, block_table, seq_lens, B)
    goes_by = dict(block_table=table, seq_lens=lens)
    if starts is not None:
        goes_by["query_start_loc"] = starts
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    elif not abs(scale) < MAX_SCALE:
        raise ValueError(f"scale must be a number below 2^127, got {scale}")
    query = query.contiguous().resolve_neg()
    if query.data_ptr() % 16:
        query = query.clone()
    fill = out is None
    if out is None:
        out = torch.empty_like(query)
    elif out.shape != query.shape or out.dtype != query.dtype or out.device != device or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError("out must be like the query: contiguous, same shape, dtype and GPU")
    elif out.is_neg():
        raise ValueError("out is negated lazily: its memory does not hold its values")
    else:
        for name, t in dict(query=query, **held, **goes_by).items():
            if overlaps(out, t):
                raise ValueError(f"out must be memory of its own, it overlaps {name}")
    longest = table.shape[-1] * PAGE_TOKENS
    # (a plan for fewer tokens may take more memory: with a workspace of its own a call is planned by what it says, as the workspace was)
    max_len = longest if max_len is None else (min(int(max_len), longest) if workspace is None else int(max_len))
    max_rows = rows if max_rows is None else int(max_rows)
    if rows == 0:
        return out
    splits = 0 if n_split is None else int(n_split)
    need = plan_bytes(cache, query.dtype, starts is not None, rows, B, Hq, max_len, max_rows, window, sinks, splits)
    if workspace is None:
        workspace = torch.empty(need // 4, dtype=torch.float32, device=device)
    else:
        check_workspace(workspace, need, device)
        for name, t in dict(query=query, out=out, **held, **goes_by).items():
            if overlaps(workspace, t):
                raise ValueError(f"the workspace overlaps {name}")
    k, v, k_scales, v_scales = cache._memory()
    with _ffi.on_device(device):
        _ffi.check(_ffi.lib().tq_attend(
            query.data_ptr(), _ffi.dtype_tag(query.dtype), rows, _ffi.ptr(starts), B, Hq, H, d, cache._tag, k, v, k_scales, v_scales,
            *cache._strides[:3], cache.num_blocks, table.data_ptr(), bt_stride, lens.data_ptr(), float(scale), max_len, max_rows, window, sinks,
            out.data_ptr(), int(fill), workspace.data_ptr(), splits, _ffi.stream_ptr(device)), "tq_attend")
    _ffi.changed(out)
    return out
