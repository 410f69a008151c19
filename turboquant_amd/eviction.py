"""Eviction from a cache by accumulated attention weight.

A sequence that has outgrown its budget keeps the tokens that mattered: the first ones, the newest ones and, of the others, those
that queries have given the most weight so far - per KV head, since heads look at different tokens.  The weights are
summed by `ExactPagedCache.add_window_weights` (a prompt) and `.decode_attention` (every token after it); `select_evictions`
says who stays and which tokens have to move, `ExactPagedCache.move_tokens` and `PagedKVPool.move_tokens` move them in the engine's
blocks and in the compressed pages of the same numbers.  (New: the reference keeps every token.)
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _ffi


def check_table(block_table: torch.Tensor, batch: int, device: torch.device) -> None:
    """What moves need of the block table of `batch` sequences whose cache lives on `device`."""
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != batch or block_table.shape[1] == 0:
        raise ValueError(f"block_table must be int32 ({batch}, max_pages)")
    _ffi.require_gpu(block_table, "block_table")
    if block_table.device != device:
        raise ValueError(f"the cache lives on {device}, block_table on {block_table.device}")


class Evictions(NamedTuple):
    """What `select_evictions` decided, for B sequences and H KV heads."""
    lens: torch.Tensor          # (B,) int32: tokens that each sequence holds from now on
    count: torch.Tensor         # (B, H) int32: moves
    dst: torch.Tensor           # (B, H, n) int32: slots that moved tokens go to, ascending, -1 from count on
    src: torch.Tensor           # (B, H, n) int32: slots that they come from
    weights: torch.Tensor       # (B, H, L) float32: of the tokens in their new slots, 0 behind them
    positions: torch.Tensor     # (B, H, L) int32: of the tokens in their new slots, of the next ones behind them
    budget: int

    def for_cache(self, block_table: torch.Tensor, num_kv_heads: int, device: torch.device):
        """(count, dst, src, table, stride of the table) for a cache of `num_kv_heads` heads on `device`."""
        B, H, _ = self.dst.shape
        if H != num_kv_heads:
            raise ValueError(f"evictions of {H} KV heads for a cache of {num_kv_heads}")
        check_table(block_table, B, device)
        if any(t.device != device for t in (self.count, self.dst, self.src)):
            raise ValueError(f"the cache lives on {device}, the evictions on {self.dst.device}")
        if self.src.shape != self.dst.shape or self.count.shape != (B, H) or any(
                t.dtype != torch.int32 or not t.is_contiguous() or t.is_neg() for t in (self.count, self.dst, self.src)):
            raise ValueError("count (B, H), dst and src (B, H, n) must be contiguous int32, as select_evictions gives them")
        table = block_table.contiguous().resolve_neg()
        return self.count, self.dst, self.src, table, table.shape[1]


def own_rows(t: torch.Tensor, twin: Optional[torch.Tensor] = None) -> bool:
    """Whether no two elements of t, the last dimension's contiguous, lie in one place; with a twin of the same strides, of both of them (one may lie in gaps that the
    other leaves)."""
    reach = t.shape[-1]
    places = [(t.stride(i), t.shape[i]) for i in range(t.dim() - 1) if t.shape[i] > 1]
    if twin is not None:
        apart = abs(twin.data_ptr() - t.data_ptr())
        if apart % t.element_size():
            return False
        places.append((apart // t.element_size(), 2))
    for stride, size in sorted(places):
        if stride < reach:
            return False
        reach = stride * (size - 1) + reach
    return True


def memory_of(t: torch.Tensor) -> Tuple[int, int]:
    """The addresses from t's first element up to behind its last."""
    first = t.data_ptr()
    return first, first + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()


def select_evictions(weights: torch.Tensor, positions: torch.Tensor, seq_lens: torch.Tensor, budget: int,
                     seen: Optional[torch.Tensor] = None, sinks: int = 4, recent: int = 0,
                     out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Evictions:
    """Cut every sequence to `budget` tokens, per KV head.

    weights (B, H, L) float32 and positions (B, H, L) int32 say of every slot how much weight its token has had and where in the
    sequence it stood; seq_lens (B,) slots are in use (L of them at most), seen (B,) tokens the sequence has had in all (None: seq_lens, nothing
    was cut before).  The first `sinks` positions and the newest `recent` always stay (sinks + recent <= budget); of the others
    the heaviest, of two alike the one in the lower slot; a NaN counts as -inf.  Sequences within the budget
    stay as they are.

    Tokens that stay and lie within the first `budget` slots do not move, those behind fill the holes in ascending order, so the slots are not
    in order of position afterwards (attention does not ask).  The inputs are left as they are; out=(weights, positions)
    takes the new ones instead of new tensors, the inputs themselves included.  The weights are numbers to choose by: neither
    gradient nor tangent goes through this call."""
    fast = _ffi.native()
    if fast is not None and out is None:
        done = fast.evict_select(weights, positions, seq_lens, seen, budget, sinks, recent)
        if done is not None:
            return Evictions(*done, budget)
    _ffi.require_gpu(weights, "weights")
    _ffi.require_gpu(positions, "positions")
    if weights.dim() != 3 or weights.shape != positions.shape or 0 in weights.shape[1:]:
        raise ValueError("weights and positions must both be (B, H, L)")
    if weights.dtype != torch.float32 or positions.dtype != torch.int32:
        raise TypeError("weights must be float32 and positions int32")
    B, H, L = weights.shape
    dev = weights.device
    if positions.device != dev:
        raise ValueError(f"weights live on {dev}, positions on {positions.device}")
    budget, sinks, recent = int(budget), int(sinks), int(recent)
    if not 1 <= budget < 1 << 31 or sinks < 0 or recent < 0 or sinks + recent > budget:
        raise ValueError(f"need 1 <= budget < 2^31 and sinks + recent <= budget, got budget {budget}, sinks {sinks}, recent {recent}")
    for name, t in (("seq_lens", seq_lens), ("seen", seen)):
        if t is not None and t.shape != (B,):
            raise ValueError(f"{name} must have one entry for each of {B} sequences")
    _ffi.require_constant("select_evictions")
    weights, positions = weights.detach().resolve_neg(), positions.resolve_neg()
    if weights.stride(2) != 1 and L > 1:
        weights = weights.contiguous()
    if positions.stride(2) != 1 and L > 1:
        positions = positions.contiguous()
    lens = seq_lens.to(device=dev, dtype=torch.int32).contiguous().resolve_neg()
    had = None if seen is None else seen.to(device=dev, dtype=torch.int32).contiguous().resolve_neg()
    if out is None:
        new_w, new_p = (torch.empty(B, H, L, dtype=t.dtype, device=dev) for t in (weights, positions))
    else:
        new_w, new_p = out
        for new, old, name in ((new_w, weights, "weights"), (new_p, positions, "positions")):
            if new.shape != old.shape or new.dtype != old.dtype or new.device != dev or (new.stride(2) != 1 and L > 1):
                raise ValueError(f"out must hold {name} (B, H, L) like the input's, slots contiguous")
            if new.is_neg():
                raise ValueError(f"out {name} is negated lazily: its memory does not hold its values")
            _ffi.require_constant("select_evictions", **{f"out {name}": new})
            if not own_rows(new):
                raise ValueError(f"out {name} must not overlap itself")
            same = new.data_ptr() == old.data_ptr() and new.stride() == old.stride()
            for other in (weights, positions):
                a, b = memory_of(new), memory_of(other)
                if not (same and other is old) and a[0] < b[1] and b[0] < a[1]:
                    raise ValueError(f"out {name} must be the input itself or memory of its own")
        a, b = memory_of(new_w), memory_of(new_p)
        if a[0] < b[1] and b[0] < a[1]:
            raise ValueError("the two tensors of out must not overlap")
    moves = max(1, min(budget, L - budget))
    whole = lambda *shape: torch.empty(*shape, dtype=torch.int32, device=dev)
    got = Evictions(whole(B), whole(B, H), whole(B, H, moves), whole(B, H, moves), new_w, new_p, budget)
    if B == 0:
        return got
    need = _ffi.lib().tq_evict_select_bytes(B, H, L, budget, moves)
    workspace = torch.empty(need // 4, dtype=torch.float32, device=dev) if need else None
    with _ffi.on_device(dev):
        _ffi.check(_ffi.lib().tq_evict_select(
            weights.data_ptr(), weights.stride(0), weights.stride(1), positions.data_ptr(), positions.stride(0), positions.stride(1),
            lens.data_ptr(), _ffi.ptr(had), B, H, L, budget, sinks, recent, moves, got.lens.data_ptr(), got.count.data_ptr(),
            got.dst.data_ptr(), got.src.data_ptr(), new_w.data_ptr(), new_w.stride(0), new_w.stride(1), new_p.data_ptr(), new_p.stride(0),
            new_p.stride(1), _ffi.ptr(workspace), _ffi.stream_ptr(dev)), "tq_evict_select")
    if out is not None:
        _ffi.changed(new_w, new_p)
    return got


def begin_rows(weights: torch.Tensor, positions: torch.Tensor, seq_lens: torch.Tensor, query_start_loc: torch.Tensor) -> None:
    """Set the rows whose sequence begins in this step - as many query rows (query_start_loc[b + 1] - query_start_loc[b]) as tokens (seq_lens[b]) - to weights 0
    and positions from 0 on, in place: a row of an engine's batch goes from one sequence to the next.  weights and positions (B, H, L) as in
    `select_evictions`; decided on the GPU, so that a captured step does it too."""
    _ffi.require_gpu(weights, "weights")
    _ffi.require_gpu(positions, "positions")
    if weights.dim() != 3 or weights.shape != positions.shape or 0 in weights.shape[1:]:
        raise ValueError("weights and positions must both be (B, H, L)")
    if weights.dtype != torch.float32 or positions.dtype != torch.int32:
        raise TypeError("weights must be float32 and positions int32")
    B, H, L = weights.shape
    dev = weights.device
    if positions.device != dev:
        raise ValueError(f"weights live on {dev}, positions on {positions.device}")
    for name, t in (("weights", weights), ("positions", positions)):
        if (t.stride(2) != 1 and L > 1) or t.is_neg() or not own_rows(t):
            raise ValueError(f"{name} need contiguous slots, memory of their own and their values in it")
        _ffi.require_constant("begin_rows", **{name: t})
    if seq_lens.shape != (B,) or query_start_loc.shape != (B + 1,):
        raise ValueError(f"seq_lens and query_start_loc must have {B} and {B + 1} entries")
    if B == 0:
        return
    lens = seq_lens.to(device=dev, dtype=torch.int32).contiguous().resolve_neg()
    starts = query_start_loc.to(device=dev, dtype=torch.int32).contiguous().resolve_neg()
    with _ffi.on_device(dev):
        _ffi.check(_ffi.lib().tq_evict_begin(
            weights.data_ptr(), weights.stride(0), weights.stride(1), positions.data_ptr(), positions.stride(0), positions.stride(1), lens.data_ptr(),
            starts.data_ptr(), B, H, L, _ffi.stream_ptr(dev)), "tq_evict_begin")
    _ffi.changed(weights, positions)
