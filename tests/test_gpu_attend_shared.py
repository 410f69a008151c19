"""Attention of steps whose sequences differ so much that the GPU shares their blocks out anew, against 64 bits.

That is where 2 to 256 sequences may see over 2048 tokens, no number of splits is given, and the longest times the number of units is more than an eighth above what
there is.  Workspaces are dirty: what a call does not write must not count."""

import math

import pytest
import torch

from tests.exact_helpers import STEP32
from tests.step_helpers import Step, half_step

pytestmark = pytest.mark.gpu

KINDS = {"bf16": (torch.bfloat16, torch.bfloat16), "fp16": (torch.float16, torch.float16), "fp8": ("fp8", torch.bfloat16), "fp8 fp16": ("fp8", torch.float16)}
UNEVEN = [61, 700, 3000, 9000]


def check(s, q, got, window=None, sinks=0, every=1):
    """Step.check's bounds, all rows of a sequence at once, every so many of them; rows behind the last sequence are not looked at.  An fp16 output of less than 2^-14
    is rounded by up to 2^-25 whatever its size."""
    scale, step, at = 1 / math.sqrt(s.d), half_step(s.dtype), 0
    G = q.shape[1] // s.H
    for b, (n, run) in enumerate(zip(s.lens, s.runs)):
        if run == 0 or n == 0:
            assert (got[at: at + run] == 0).all()
            at += run
            continue
        pick = torch.arange(run)[(torch.arange(run) % every == 0) | (torch.arange(run) == run - 1)]
        k, v, there = (x.to(s.device) for x in s.tokens(b, n))
        p, t = (n - run + pick).to(s.device)[:, None], torch.arange(n, device=s.device)
        seen = there & (t <= p)
        if window is not None:
            seen &= (t > p - window) | (t < sinks)
        seen = seen.repeat_interleave(G, 0)
        for h in range(s.H):
            x = q[at + pick, h * G: (h + 1) * G].double().reshape(-1, s.d).to(s.device)
            kh, vh = k[:, h].contiguous(), v[:, h].contiguous()
            some = seen.any(1, keepdim=True)
            w = torch.softmax((x @ kh.T.contiguous() * scale).masked_fill(~seen, -math.inf), -1).masked_fill(~some, 0)
            out, size = w @ vh, w @ vh.abs()
            score = (s.d + 4) * STEP32 * (x.abs() @ kh.abs().T.contiguous() * scale).masked_fill(~seen, 0).amax(1, keepdim=True)
            err = (2 * score + (n + 64) * STEP32 + 1.01 * step) * size
            mine = got[(at + pick).to(got.device), h * G: (h + 1) * G].reshape(-1, s.d).double()
            assert torch.isfinite(mine).all(), f"sequence {b} of {n}: not finite"
            off, allowed = (mine - out).abs(), err + step * (out.abs() + err) + (2.0 ** -25 if s.dtype == torch.float16 else 1e-30)
            assert (off <= allowed).all(), f"sequence {b} of {n}, head {h}: off by {float((off / allowed).max()):.3g} of what is allowed"
        at += run


def dirty(work, i):
    """Old contents of a workspace: NaN, or any bytes."""
    if i % 2:
        work.fill_(math.nan)
    else:
        g = torch.Generator(device=work.device).manual_seed(i)
        work.view(torch.int32).copy_(torch.randint(-(1 << 31), (1 << 31) - 1, (work.numel(),), generator=g, device=work.device, dtype=torch.int64).to(torch.int32))
    return work


def workspace(cache, kind, dtype, rows, Hq, **kw):
    return cache.workspace(rows, Hq, dtype=dtype, **kw) if kind.startswith("fp8") else cache.step_workspace(rows, Hq, **kw)


def steps(s, Hq, kind, window=None, sinks=0, max_len=None, max_rows=None, decode=False, every=1, extra=0):
    """The step with no workspace, and with dirty ones, an output given or not: right, and the same bits."""
    q = s.query(Hq)
    x, cache = q.to(s.device), s.cache()
    longest, most = s.table.shape[1] * 16 if max_len is None else max_len, max_rows or s.rows
    seen = dict(window=window, sinks=sinks)
    if decode:
        call = lambda **kw: cache.decode_attention(x, s.table, s.seq_lens, max_len=longest, **seen, **kw)
        room = dict(max_len=longest, **seen)
    else:
        call = lambda **kw: cache.attention(x, s.starts, s.table, s.seq_lens, max_len=longest, max_rows=most, **seen, **kw)
        room = dict(max_len=longest, B=len(s.lens), max_rows=most, **seen)
    first = None
    for i in range(3):
        work = dirty(workspace(cache, kind, q.dtype, s.rows, Hq, **room), i)
        got = call(workspace=work)
        if first is None:
            first = got
            check(s, q, got, window, sinks, every)
        assert torch.equal(got, first)
        out = torch.full_like(x, 5)
        call(workspace=dirty(work, i + 1), out=out)
        n = s.rows - s.extra
        assert torch.equal(out[:n], first[:n]) and (out[n:] == 5).all() and (got[n:] == 0).all()
    assert torch.equal(call(), first)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("runs", [[1, 2, 1, 3], [40, 1, 20, 9]])
def test_lengths_that_differ(gpu, kind, d, runs):
    """Few rows and many; with and without rows of no sequence; windows that see over 2048 tokens."""
    s = Step(UNEVEN, runs, 2, d, *KINDS[kind], extra=13)
    most = max(runs)
    steps(s, 8, kind, max_rows=most)
    steps(s, 8, kind, 2500, 7, max_rows=most)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("G", [1, 7, 20, 40])
def test_single_tokens(gpu, kind, d, G):
    s = Step(UNEVEN, [1] * 4, 2, d, *KINDS[kind])
    if kind.startswith("fp8"):
        steps(s, 2 * G, kind, decode=True)
    steps(s, 2 * G, kind, 3000, 3, decode=True)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("more", [3, 254, 255, 256])
@pytest.mark.parametrize("rows", [1, 3])
def test_one_among_short_ones(gpu, kind, more, rows):
    """Up to 256 sequences are looked at together, and from 257 on shared out as planned."""
    lens = [1 + (7 * i) % 40 for i in range(more)]
    lens.insert(more // 2, 2500)
    steps(Step(lens, [min(n, rows) for n in lens], 1, 64, *KINDS[kind], extra=5), 4, kind, max_rows=rows)
    steps(Step(lens, [0 if i % 3 == 0 else min(n, rows) for i, n in enumerate(lens)], 1, 64, *KINDS[kind], width=500), 4, kind, 2200, 1)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("far", [20000, 200000])
def test_planned_for_far_more(gpu, kind, far):
    """max_len by far above the lengths: more splits than there are blocks for."""
    for runs in ([1, 1, 2], [33, 2, 50]):
        steps(Step([300, 2600, 70], runs, 2, 64, *KINDS[kind], width=far // 16, extra=1), 8, kind, max_len=far, max_rows=max(runs))


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("rows", [15, 16])
def test_rows_around_512(gpu, kind, rows):
    """480 and 512 rows x heads: joined by workgroups or by wavefronts, up to 1024, 96 or 64 shares of a row."""
    steps(Step([16000, 90, 40], [rows - 2, 1, 1], 1, 128, *KINDS[kind]), 32, kind, max_rows=rows - 2)
    steps(Step([16000, 90, 40], [1, 1, rows - 2], 1, 128, *KINDS[kind]), 32, kind, max_rows=1)


@pytest.mark.parametrize("kind", ["bf16", "fp8 fp16"])
def test_rows_of_several_a_wavefront(gpu, kind):
    """32768 rows x heads: the join looks at several rows a wavefront, one sequence's are split."""
    s = Step([6000, 40, 1000, 9], [100, 40, 876, 8], 1, 64, *KINDS[kind], extra=3)
    steps(s, 32, kind, max_rows=876, every=37)


@pytest.mark.parametrize("kind", list(KINDS))
def test_captured_and_replayed_as_other_steps(gpu, kind):
    """One graph: lengths that are alike (as planned) and that differ (shared out anew), in turn."""
    s = Step(UNEVEN, [1, 2, 1, 3], 2, 128, *KINDS[kind])
    q, cache = s.query(8), s.cache()
    x = q.to(gpu)
    call = lambda: cache.attention(x, s.starts, s.table, s.seq_lens, max_len=9008, max_rows=3)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for lens in (UNEVEN, [61, 60, 61, 61], [2, 700, 1, 8999], [9, 3, 2900, 5], UNEVEN):
        s.lens = lens
        s.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call())
        check(s, q, out)
