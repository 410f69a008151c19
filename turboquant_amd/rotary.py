"""What is in front of a cache in every step: the norm of each head of queries and keys, and their rotation by position.

(New: the reference gets its keys rotated from the engine's model.)
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _ffi
from .attend import overlaps, row_strides
from .eviction import own_rows

MAX_HEAD_DIM = 512


def inverse_frequencies(rotary_dim: int, theta: float = 10000.0, device=None) -> torch.Tensor:
    """theta ** (-2 i / rotary_dim) for i < rotary_dim / 2, in float64 as `rotate_heads` takes them."""
    return theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)


def rotate_heads(query: torch.Tensor, key: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False,
                 out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """query (rows, Hq, d) and key (rows, H_kv, d), fp32, fp16 or bf16, normed head by head and rotated by positions (rows,) int32 or int64.

    With q_weight / k_weight (d,) a head x becomes x / sqrt(mean x^2 + eps) * weight; without, it stays.  Then the pairs (i, i + r / 2) of its first
    r = 2 len(inv_freq) channels, or (2 i, 2 i + 1) if interleaved, turn by the angle position * inv_freq[i] (float64, `inverse_frequencies`), which is
    as good at position 2^20 as at 1.  All of it in 32 bits, rounded once.  Views of a fused projection are read where they are.

    Returns new contiguous tensors, or out=(query, key), channels contiguous: each may be its own input (not the other, nor memory that the
    other shares)."""
    fast = _ffi.native()
    if fast is not None and out is None:
        done = fast.rotate(query, key, positions, inv_freq, q_weight, k_weight, eps, interleaved)
        if done is not None:
            return done
    _ffi.require_gpu(query, "query")
    _ffi.require_gpu(key, "key")
    if query.dim() != 3 or key.dim() != 3 or query.shape[0] != key.shape[0] or query.shape[2] != key.shape[2]:
        raise ValueError("query must be (rows, Hq, d) and key (rows, H_kv, d)")
    rows, Hq, d = query.shape
    H, dev, tag = key.shape[1], query.device, _ffi.dtype_tag(query.dtype)
    if key.dtype != query.dtype or key.device != dev:
        raise TypeError("query and key must have one dtype and live on one GPU")
    if d == 0 or d % 8 or d > MAX_HEAD_DIM or Hq + H == 0:
        raise ValueError(f"head_dim must be a multiple of 8 up to {MAX_HEAD_DIM}, got {Hq} and {H} heads of {d}")
    if positions.shape != (rows,) or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions must be int32 or int64 ({rows},)")
    r = 2 * inv_freq.shape[0] if inv_freq.dim() == 1 else -1
    if inv_freq.dtype != torch.float64 or r < 0 or r % 8 or r > d:
        raise ValueError(f"inv_freq must be float64, one for each of up to {d // 2} pairs, a multiple of 4 of them")
    for name, t in (("positions", positions), ("inv_freq", inv_freq)):
        _ffi.require_gpu(t, name)
        if t.device != dev:
            raise ValueError(f"{name} lives on {t.device}, the query on {dev}")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (w.shape != (d,) or w.dtype != query.dtype or w.device != dev):
            raise ValueError(f"{name} must be ({d},) like the query: same dtype and GPU")
    _ffi.require_constant("rotate_heads", query=query, key=key, q_weight=q_weight, k_weight=k_weight, inv_freq=inv_freq)
    align = 16 if query.dtype == torch.float32 else 8
    fits = lambda t: t.stride(2) == 1 and all(s % 4 == 0 for s in row_strides(t)) and t.data_ptr() % align == 0
    given = query, key
    query, key = (t if fits(t) else t.contiguous() for t in (query.resolve_neg(), key.resolve_neg()))
    query, key = (t if fits(t) else t.clone() for t in (query, key))
    if out is None:
        new = tuple(torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (query, key))
    else:
        new = tuple(out)
        if len(new) != 2:
            raise ValueError("out must be two tensors, for query and key")
        for t, old, other, name in zip(new, given, given[::-1], ("query", "key")):
            if t.shape != old.shape or t.dtype != old.dtype or t.device != dev or not fits(t) or t.is_neg():
                raise ValueError(f"out {name} must be like it: same shape, dtype and GPU, channels contiguous, rows on {align}-byte boundaries")
            _ffi.require_constant("rotate_heads", **{f"out {name}": t})
            if not own_rows(t):
                raise ValueError(f"out {name} must not overlap itself")
            # (a head is read by the lanes that write it: over its own input only, and the other input's heads are read at other times)
            itself = t.data_ptr() == old.data_ptr() and row_strides(t) == row_strides(old)
            if any(overlaps(t, x) and not _beside(t, x) for x in ((other,) if itself else (old, other))):
                raise ValueError(f"out {name} must be {name} itself or memory of its own")
            for what, x in (("positions", positions), ("inv_freq", inv_freq), ("q_weight", q_weight), ("k_weight", k_weight)):
                if x is not None and overlaps(t, x):
                    raise ValueError(f"out {name} overlaps {what}")
        if overlaps(*new) and not _beside(*new):
            raise ValueError("the two tensors of out must not overlap")
    q_weight, k_weight = (None if w is None else _weight(w, align) for w in (q_weight, k_weight))
    positions, inv_freq = positions.contiguous().resolve_neg(), inv_freq.contiguous().resolve_neg()
    if rows == 0:
        return new
    with _ffi.on_device(dev):
        _ffi.check(_ffi.lib().tq_rotate_heads(
            query.data_ptr(), key.data_ptr(), tag, rows, Hq, H, d, *row_strides(query), *row_strides(key), positions.data_ptr(),
            int(positions.dtype == torch.int64), inv_freq.data_ptr(), r, int(bool(interleaved)), _ffi.ptr(q_weight), _ffi.ptr(k_weight), float(eps),
            new[0].data_ptr(), *row_strides(new[0]), new[1].data_ptr(), *row_strides(new[1]), _ffi.stream_ptr(dev)), "tq_rotate_heads")
    if out is not None:
        _ffi.changed(*new)
    return new


def _weight(w: torch.Tensor, align: int) -> torch.Tensor:
    w = w.contiguous().resolve_neg()
    return w.clone() if w.data_ptr() % align else w


def _beside(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether a and b are columns of one matrix of rows that share none: views of a fused projection."""
    step = a.stride(0)
    if step != b.stride(0) or a.element_size() != b.element_size():
        return False
    size = a.element_size()
    first = min(a.data_ptr(), b.data_ptr())
    (x, nx), (y, ny) = (((t.data_ptr() - first) // size, (t.shape[1] - 1) * t.stride(1) + t.shape[2]) for t in (a, b))
    return x + nx <= step and y + ny <= step and (x + nx <= y or y + ny <= x)
