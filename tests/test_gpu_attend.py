"""Attention of a step's rows over exact blocks and over the 8-bit cache, with and without a window, against 64 bits."""

import math

import pytest
import torch

from tests.step_helpers import Step

pytestmark = pytest.mark.gpu

KINDS = {"bf16": (torch.bfloat16, torch.bfloat16), "fp16": (torch.float16, torch.float16), "fp8": ("fp8", torch.bfloat16), "fp8 fp16": ("fp8", torch.float16)}


def make(kind, lens, runs, H, d, **kw):
    return Step(lens, runs, H, d, *KINDS[kind], **kw)


def run(s, Hq, window=None, sinks=0, scale=None, **kw):
    q = s.query(Hq, **{k: kw.pop(k) for k in ("size",) if k in kw})
    got = s.cache().attention(q.to(s.device), s.starts, s.table, s.seq_lens, scale=scale, window=window, sinks=sinks, **kw)
    s.check(q, got, 1 / math.sqrt(s.d) if scale is None else scale, window, sinks)
    return q, got


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("Hq,H", [(4, 2), (5, 1), (16, 1), (24, 2)])
def test_single_tokens(gpu, kind, d, Hq, H):
    lens = [1, 16, 17, 100, 0, 333]
    s = make(kind, lens, [1] * 6, H, d)
    q = s.query(Hq)
    for window, sinks in ((None, 0), (1, 0), (20, 3), (1000, 1000)):
        got = s.cache().decode_attention(q.to(gpu), s.table, s.seq_lens, window=window, sinks=sinks)
        if window is None and kind in ("bf16", "fp16"):
            got = s.cache().attention(q.to(gpu), s.starts, s.table, s.seq_lens)
        s.check(q, got, 1 / math.sqrt(d), window, sinks)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("window,sinks", [(None, 0), (7, 0), (33, 5), (64, 70)])
def test_rows_of_several_lengths(gpu, kind, d, window, sinks):
    run(make(kind, [3, 70, 17, 130, 5, 40], [3, 2, 17, 37, 0, 1], 2, d), 6, window, sinks)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("G", [1, 3, 8, 32])
@pytest.mark.parametrize("runs", [[2, 1], [5, 3], [70, 20]])
def test_heads_on_one(gpu, kind, G, runs):
    run(make(kind, [90, 20], runs, 1, 128), G)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("n_split", [1, 2, 5, 16, 17, 40])
def test_splits(gpu, kind, n_split):
    for runs in ([1, 1, 1], [4, 1, 7]):
        run(make(kind, [1300, 10, 601], runs, 1, 128), 4, n_split=n_split)
        run(make(kind, [1300, 10, 601], runs, 1, 128), 4, 200, 17, n_split=n_split)


@pytest.mark.parametrize("kind", list(KINDS))
def test_longer_than_planned_for(gpu, kind):
    """max_len and max_rows are for the plan: what exceeds them is right, too."""
    s = make(kind, [900, 333], [40, 9], 2, 64)
    run(s, 4, max_len=16, max_rows=1)
    run(s, 4, 100, 2, max_len=16, max_rows=1)


@pytest.mark.parametrize("kind", list(KINDS))
def test_rows_of_no_sequence_and_rows_without_tokens(gpu, kind):
    s = make(kind, [3, 20, 0], [5, 2, 2], 2, 64, extra=11)
    for n_split in (1, 3):
        q, got = run(s, 4, n_split=n_split)
        assert (got[:2] == 0).all() and (got[7:] == 0).all()
        out = torch.full_like(got, 5.0)
        assert s.cache().attention(q.to(gpu), s.starts, s.table, s.seq_lens, out=out, n_split=n_split) is out
        assert (out[9:] == 5).all() and torch.equal(out[:9], got[:9])
    none = torch.zeros(1, dtype=torch.int32, device=gpu)
    empty = s.cache().attention(q.to(gpu), none, s.table[0], s.seq_lens[:0])
    assert (empty == 0).all() and empty.shape == q.shape


@pytest.mark.parametrize("kind", list(KINDS))
def test_tables(gpu, kind):
    """Blocks outside the cache have no weight, lengths beyond the table end with it; one table for all."""
    s = make(kind, [100, 60, 50], [1, 3, 2], 1, 64)
    s.table_cpu[0, 2], s.table_cpu[1, 3], s.table_cpu[2, 0] = -1, s.blocks, 1 << 30
    s.table = s.table_cpu.to(gpu)
    run(s, 3)
    run(s, 3, 40, 4, n_split=3)
    s.width = 3
    s.table_cpu = s.table_cpu[:, :3].contiguous()
    s.table = s.table_cpu.to(gpu)
    run(s, 3)
    one = make(kind, [70], [2], 1, 64)
    q = one.query(2)
    a = one.cache().attention(q.to(gpu), one.starts, one.table, one.seq_lens)
    assert torch.equal(a, one.cache().attention(q.to(gpu), one.starts, one.table[0], one.seq_lens))


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("layout", ["heads", "padded"])
def test_blocks_of_other_layouts(gpu, kind, layout):
    run(make(kind, [100, 33], [20, 1], 2, 128, layout=layout), 4, 50, 3)


@pytest.mark.parametrize("kind", list(KINDS))
def test_large_scores_and_scales(gpu, kind):
    """One token has all the weight; negative and zero scales."""
    s = make(kind, [300, 40], [1, 9], 1, 64)
    run(s, 2, size=30.0)
    run(make(kind, [200, 90], [70, 3], 1, 64), 4, scale=-0.3)
    run(make(kind, [200, 90], [70, 3], 1, 64), 4, scale=0.0)
    run(s, 2, scale=-0.2)
    run(s, 2, scale=0.0)


@pytest.mark.parametrize("kind", list(KINDS))
def test_many_sequences(gpu, kind):
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 60, (300,), generator=g).tolist()
    runs = [min(n, int(r)) for n, r in zip(lens, torch.randint(0, 6, (300,), generator=g))]
    run(make(kind, lens, runs, 1, 64), 2)


def step_graph(s, q, call):
    graph = torch.cuda.CUDAGraph()
    call()
    with torch.cuda.graph(graph):
        out = call()
    return graph, out


@pytest.mark.parametrize("kind", list(KINDS))
def test_captured_with_workspaces_of_their_own(gpu, kind):
    s = make(kind, [700, 90], [1, 1], 2, 128)
    q = s.query(8).to(gpu)
    cache = s.cache()
    work = cache.step_workspace if kind in ("bf16", "fp16") else cache.workspace
    spaces = [work(2, 8, 800, window=300, sinks=4, **({} if kind in ("bf16", "fp16") else dict(dtype=q.dtype))) for _ in range(2)]
    outs = [torch.empty_like(q) for _ in range(2)]
    calls = [lambda w=w, o=o: cache.decode_attention(q, s.table, s.seq_lens, window=300, sinks=4, workspace=w, out=o, max_len=800) for w, o in zip(spaces, outs)]
    graphs = [step_graph(s, q, c)[0] for c in calls]
    sides = [torch.cuda.Stream() for _ in range(2)]
    for i in range(3):
        q.copy_(s.query(8, seed=10 + i))
        torch.cuda.synchronize()
        for graph, side in zip(graphs, sides):
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        want = cache.decode_attention(q, s.table, s.seq_lens, window=300, sinks=4, max_len=800)
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
        s.check(q.cpu(), want, 1 / math.sqrt(128), 300, 4)


@pytest.mark.parametrize("kind", list(KINDS))
def test_results_repeat_and_depend_on_nobody_else(gpu, kind):
    """The same call twice, and a sequence alone or beside others with the same plan, give the same bits."""
    s = make(kind, [500, 40, 77], [3, 1, 20], 2, 64)
    q = s.query(6).to(gpu)
    a = s.cache().attention(q, s.starts, s.table, s.seq_lens, n_split=3, max_rows=20)
    assert torch.equal(a, s.cache().attention(q, s.starts, s.table, s.seq_lens, n_split=3, max_rows=20))
    alone = s.cache().attention(q[:3], s.starts[:2], s.table[:1], s.seq_lens[:1], n_split=3, max_rows=20, max_len=s.table.shape[1] * 16)
    assert torch.equal(a[:3], alone) or (a[:3] - alone).abs().max() <= 2 ** -7 * alone.abs().max()


@pytest.mark.parametrize("kind", list(KINDS))
def test_strided_queries_and_inference(gpu, kind):
    s = make(kind, [50, 20], [4, 1], 1, 64)
    q = s.query(3)
    wide = torch.cat([q, q], -1).to(gpu)[..., :64]
    with torch.inference_mode():
        s.check(q, s.cache().attention(wide, s.starts.long(), s.table, s.seq_lens.cpu()), 0.125)
        s.check(q, s.cache().attention(torch._neg_view(-q.to(gpu)), s.starts, s.table, s.seq_lens), 0.125)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("G,runs", [(1, [1, 1]), (4, [3, 5]), (4, [60, 37]), (128, [2, 1]), (160, [3, 2])])
@pytest.mark.parametrize("window,sinks", [(None, 0), (21, 6)])
def test_values_that_are_not_finite(gpu, kind, d, G, runs, window, sinks):
    """Infinities and NaN among the values: in the channels of the rows that see them, and nowhere else."""
    lens = [130, 90]
    s = make(kind, lens, runs, 2, d)
    q = s.query(2 * G).to(gpu)
    kw = dict(window=window, sinks=sinks)
    inf, nan = float("inf"), float("nan")
    put = []                                                 # (sequence, token, head, channel, value)
    for b, n in enumerate(lens):
        edge = [n - 1, n - 2, n - runs[b], n - runs[b] + 1, n - runs[b] - 20, n - 22, n - 21, n - 20, 0, 5, 6, 33, 64]
        for i, t in enumerate(e for e in edge if 0 <= e < n):
            put.append((b, t, i % 2, (7 * i + b) % d, nan if kind.startswith("fp8") else (inf, -inf, nan)[i % 3]))
            put.append((b, t, 1, d - 1, nan if kind.startswith("fp8") else inf))
    odd = torch.zeros(2, max(lens), 2, d)
    for b, t, h, c, x in put:
        where = (int(s.table_cpu[b, t // 16]), t % 16, h, c)
        s.q[1].view(torch.uint8 if kind.startswith("fp8") else s.q[1].dtype)[where] = 0
        s.v64[where] = 0
        odd[b, t, h, c] = x
    clean = s.cache().attention(q, s.starts, s.table, s.seq_lens, **kw)
    s.check(q.cpu(), clean, 1 / math.sqrt(d), window, sinks)
    for b, t, h, c, x in put:
        s.q[1].view(torch.uint8 if kind.startswith("fp8") else s.q[1].dtype)[int(s.table_cpu[b, t // 16]), t % 16, h, c] = 0x7f if kind.startswith("fp8") else x
    for n_split in (None, 1, 3):
        got = s.cache().attention(q, s.starts, s.table, s.seq_lens, **kw, **({} if n_split is None else {"n_split": n_split})).cpu()
        at = 0
        for b, run in enumerate(runs):
            for i in range(run):
                p = lens[b] - run + i
                t = torch.arange(p + 1)
                seen = (t > p - window) | (t < sinks) if window else torch.ones(p + 1, dtype=torch.bool)
                add = odd[b, : p + 1][seen].sum(0).repeat_interleave(G, 0)
                assert torch.equal(got[at + i].isfinite(), add.isfinite()), (b, i)
                assert torch.equal(got[at + i].isposinf(), add.isposinf()) and torch.equal(got[at + i].isneginf(), add.isneginf()), (b, i)
            at += run
        if n_split is None:
            assert torch.equal(torch.where(got.isfinite(), got, clean.cpu()), clean.cpu())
