"""Eviction: who stays, the lists of moves, and the moves in exact and compressed pages.  Everything is held to equality."""

import math

import pytest
import torch

from tests.exact_helpers import DTYPES, PAGE, Sequences, evict64

pytestmark = pytest.mark.gpu


def weights_of(B, H, L, seed, kind="sums"):
    g = torch.Generator().manual_seed(seed)
    w = torch.exp(2 * torch.randn(B, H, L, generator=g))
    if kind == "ties":
        w = torch.randint(0, 3, (B, H, L), generator=g).float()
    elif kind == "equal":
        w = torch.full((B, H, L), 0.25)
    elif kind == "odd":
        odd = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, -1.0, 1e-45, 3.4028234663852886e38, -3.4e38])
        w = odd[torch.randint(0, len(odd), (B, H, L), generator=g)]
    elif kind == "close":                       # neighbours in the last bits
        w = (torch.randint(0, 2000, (B, H, L), generator=g).int() + 0x3f800000).view(torch.float32)
    return w


def check(w, pos, lens, budget, seen=None, sinks=4, recent=0, out=None):
    from turboquant_amd.eviction import select_evictions
    gpu = torch.device("cuda:0")
    to = lambda t: None if t is None else t.to(gpu)
    w_d, p_d = to(w), to(pos)
    lens_t = torch.tensor(lens, dtype=torch.int32)
    seen_t = None if seen is None else torch.tensor(seen, dtype=torch.int32)
    e = select_evictions(w_d, p_d, to(lens_t), budget, seen=to(seen_t), sinks=sinks, recent=recent, out=(w_d, p_d) if out == "inputs" else None)
    want = evict64(w, pos, lens_t, seen_t, budget, sinks, recent)
    for name, got, t in zip(("lens", "count", "dst", "src", "weights", "positions"), e, want):
        g = got.cpu()
        if name == "weights":
            g, t = g.view(torch.int32), t.view(torch.int32)
        assert torch.equal(g, t), name
    if out is None:
        assert torch.equal(w_d.cpu().view(torch.int32), w.view(torch.int32)) and torch.equal(p_d.cpu(), pos)
    else:
        assert e.weights is w_d or e.weights.data_ptr() == w_d.data_ptr()
    return e


def in_order(B, H, L):
    return torch.arange(L, dtype=torch.int32).expand(B, H, L).contiguous()


@pytest.mark.parametrize("kind", ["sums", "ties", "equal", "odd", "close"])
@pytest.mark.parametrize("L,budget", [(1, 1), (2, 1), (17, 16), (100, 33), (1000, 999), (1025, 512), (3000, 7), (5000, 2048)])
def test_who_stays(gpu, L, budget, kind):
    w, pos = weights_of(2, 3, L, L, kind), in_order(2, 3, L)
    for sinks, recent in ((0, 0), (min(4, budget), 0), (budget // 4, budget // 2), (0, budget)):
        check(w, pos, [L, max(0, L - 1)], budget, sinks=sinks, recent=recent)


@pytest.mark.parametrize("L,budget", [(40000, 1000), (131072, 16384), (150001, 75000), (700001, 20000), (700001, 650000)])
def test_long_rows(gpu, L, budget):
    for kind in ("sums", "ties", "close"):
        check(weights_of(1, 2, L, 1, kind), in_order(1, 2, L), [L - 3], budget, sinks=16, recent=100, out="inputs" if kind == "ties" else None)


@pytest.mark.parametrize("L,budget", [(16384, 5), (16385, 5), (16385, 16384), (4096, 4095), (4097, 100), (32769, 32768), (33000, 8192), (50000, 8193), (40000, 20000)])
def test_rows_at_the_ends_of_their_parts(gpu, L, budget):
    """One workgroup and several, budgets at and off a part's end, and rows of a batch that are within the budget beside others."""
    for kind, sinks, recent in (("sums", 0, 0), ("equal", min(4, budget), 0), ("odd", 0, min(budget, 1000))):
        w, pos = weights_of(3, 1, L, budget, kind), in_order(3, 1, L)
        check(w, pos, [L, min(L, budget + 1), budget - 1], budget, sinks=sinks, recent=recent, out="inputs" if kind == "equal" else None)


def test_lengths_within_the_budget_and_of_nothing(gpu):
    w, pos = weights_of(6, 2, 64, 3), in_order(6, 2, 64)
    e = check(w, pos, [0, 1, 31, 32, 33, 64], 32, sinks=1, recent=2)
    assert e.lens.tolist() == [0, 1, 31, 32, 32, 32]
    check(w, pos, [-4, 100, 2 ** 31 - 1, -2 ** 31, 64, 5], 32, seen=[0, 100, 70, 0, 64, 5])
    check(w, pos, [64] * 6, 64)
    check(w, pos, [64] * 6, 1000)


@pytest.mark.parametrize("out", [None, "inputs"])
def test_cut_again_and_again(gpu, out):
    """A budget kept up over many tokens: positions out of order, few moves a time."""
    B, H, L, budget = 3, 2, 120, 100
    w, pos = weights_of(B, H, L, 4), in_order(B, H, L)
    lens, seen = [110, 60, 120], [110, 60, 120]
    g = torch.Generator().manual_seed(1)
    for _ in range(6):
        e = check(w, pos, lens, budget, seen=seen, sinks=2, recent=30, out=out)
        w, pos, held = e.weights.cpu(), e.positions.cpu(), e.lens.tolist()
        new = [7, 20, 1]
        lens, seen = [n + k for n, k in zip(held, new)], [s + k for s, k in zip(seen, new)]
        w += torch.rand(B, H, L, generator=g) * (torch.arange(L) < torch.tensor(lens)[:, None, None])
        for b in range(B):
            for h in range(H):
                now = pos[b, h, : lens[b]].tolist()
                assert len(set(now)) == lens[b] and all(p in now for p in range(seen[b] - new[b], seen[b]))


def test_positions_that_are_not_a_sequence_s(gpu):
    """Whatever the positions say - all protected, none, the extremes of int32 - `budget` of them stay."""
    w = weights_of(1, 4, 90, 2)
    pos = torch.stack([torch.zeros(90), torch.full((90,), 50), torch.full((90,), -2.0 ** 31), torch.full((90,), 2.0 ** 31 - 1)])
    pos = pos.double().to(torch.int64).clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32)[None]
    check(w, pos.contiguous(), [90], 40, seen=[60], sinks=4, recent=10)


def test_strided_inputs_and_outputs(gpu):
    from turboquant_amd.eviction import select_evictions
    w, pos = weights_of(2, 3, 50, 8), in_order(2, 3, 50)
    want = evict64(w, pos, torch.tensor([50, 44]), None, 20, 4, 3)
    lens = torch.tensor([50, 44], dtype=torch.int32, device=gpu)
    wide_w, wide_p = torch.zeros(3, 2, 60, device=gpu), torch.zeros(3, 2, 60, dtype=torch.int32, device=gpu)
    w_d, p_d = wide_w.transpose(0, 1)[..., 5:55], wide_p.transpose(0, 1)[..., 5:55]
    w_d.copy_(w)
    p_d.copy_(pos)
    for out in (None, (w_d, p_d)):
        e = select_evictions(w_d, p_d, lens, 20, recent=3, out=out)
        for got, t in zip(e, want):
            assert torch.equal(got.cpu(), t)
    assert not wide_w[..., :5].any() and not wide_w[..., 55:].any() and not wide_p[..., 55:].any()
    # slots that are not neighbours are read too
    w2 = torch.stack([w, w], -1).to(gpu)[..., 0]
    assert torch.equal(select_evictions(w2, pos.to(gpu), lens, 20, recent=3).dst.cpu(), want[2])


@pytest.mark.parametrize("layout", ["engine", "heads", "padded"])
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("fp16", 64), ("fp32", 192), ("bf16", 576)])
def test_moves_in_the_exact_cache(gpu, dtype, d, layout):
    from turboquant_amd.eviction import select_evictions
    from turboquant_amd.exact import ExactPagedCache
    seqs = Sequences([300, 20, 111], 3, d, DTYPES[dtype], layout=layout)
    w, pos = weights_of(3, 3, 300, d).to(gpu), in_order(3, 3, 300).to(gpu)
    seqs.table[0, 2] = -1                                       # a page that is not there: its tokens move nowhere
    e = select_evictions(w, pos, seqs.seq_lens, 100, recent=40)
    want = seqs.kv.clone().cpu()
    table, dst, src = seqs.table.cpu(), e.dst.cpu(), e.src.cpu()
    for b in range(3):
        for h in range(3):
            for n in range(int(e.count[b, h])):
                to, of = int(dst[b, h, n]), int(src[b, h, n])
                if table[b, to // PAGE] < 0 or table[b, of // PAGE] < 0:
                    continue
                want[:, table[b, to // PAGE], to % PAGE, h] = want[:, table[b, of // PAGE], of % PAGE, h]
    ExactPagedCache.from_engine(seqs.kv).move_tokens(e, seqs.table)
    bits = torch.int32 if dtype == "fp32" else torch.int16
    assert torch.equal(seqs.kv.cpu().contiguous().view(bits), want.contiguous().view(bits))


@pytest.mark.parametrize("d,key_bits,value_bits,group,dtype", [
    (128, 3, 2, 32, "bf16"), (128, 3, 4, 32, "bf16"), (128, 4, 8, 32, "fp16"), (64, 2, 4, 32, "bf16"), (256, 3, 2, 64, "fp16"),
    (576, 4, 4, 32, "bf16"), (192, 3, 4, 32, "fp32"), (320, 5, 2, 64, "bf16")])
def test_moves_in_the_compressed_pages(gpu, d, key_bits, value_bits, group, dtype):
    """Every token's codes, norms and scales arrive as they were; nothing else in any page changes."""
    from turboquant_amd.eviction import select_evictions
    from turboquant_amd.paged import PagedKVPool
    from turboquant_amd.quantizer import TurboQuantProd
    B, N, H, budget = 2, 150, 2, 70
    pool = PagedKVPool(TurboQuantProd(d, bits=key_bits, device=gpu), H, 25, value_bits=value_bits, value_group_size=group, dtype=DTYPES[dtype])
    pages = (N + PAGE - 1) // PAGE
    table = torch.randperm(25, generator=torch.Generator().manual_seed(0))[: B * pages].view(B, pages).to(torch.int32).to(gpu)
    g = torch.Generator().manual_seed(d)
    k, v = (torch.randn(B, N, H, d, generator=g).to(DTYPES[dtype]).to(gpu) for _ in range(2))
    pool.append(k, v, table)
    before, was = [pool.export_flat(table[b], N) for b in range(B)], pool.data.clone()
    w, pos = weights_of(B, H, N, d).to(gpu), in_order(B, H, N).to(gpu)
    e = select_evictions(w, pos, torch.tensor([N, N - 31], dtype=torch.int32, device=gpu), budget, recent=20)
    pool.move_tokens(e, table)
    assert int(e.count.min()) > 5
    for b in range(B):
        after = pool.export_flat(table[b], N)
        for h in range(H):
            n = int(e.count[b, h])
            of = torch.arange(N)
            of[e.dst[b, h, :n].cpu().long()] = e.src[b, h, :n].cpu().long()
            for x, y in zip(before[b], after):
                assert torch.equal(x[h].cpu()[of], y[h].cpu())
    # pages without holes, pages of nobody
    others = [p for p in range(25) if p not in table.cpu()[:, : (budget + PAGE - 1) // PAGE]]
    assert torch.equal(pool.data[others], was[others])


def test_compressed_moves_over_bad_pages(gpu):
    from turboquant_amd.eviction import select_evictions
    from turboquant_amd.paged import PagedKVPool
    from turboquant_amd.quantizer import TurboQuantProd
    pool = PagedKVPool(TurboQuantProd(64, bits=3, device=gpu), 1, 8, dtype=torch.bfloat16)
    table = torch.arange(8, dtype=torch.int32, device=gpu)[None]
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(1, 128, 1, 64, generator=g).bfloat16().to(gpu) for _ in range(2))
    pool.append(k, v, table)
    before = pool.export_flat(table[0], 128)
    e = select_evictions(weights_of(1, 1, 128, 0).to(gpu), in_order(1, 1, 128).to(gpu), torch.tensor([128], device=gpu), 64)
    bad = table.clone()
    bad[0, 1], bad[0, 6] = 8, -1
    pool.move_tokens(e, bad)
    of = torch.arange(128)
    for to, s in zip(e.dst[0, 0].tolist(), e.src[0, 0].tolist()):
        if to >= 0 and to // PAGE != 1 and s // PAGE != 6:
            of[to] = s
    for x, y in zip(before, pool.export_flat(table[0], 128)):
        assert torch.equal(x[0].cpu()[of], y[0].cpu())
    short = table[:, :3].contiguous()                         # a row that ends before the sources: nothing moves
    was = pool.data.clone()
    pool.move_tokens(e, short)
    assert torch.equal(pool.data, was)


def test_graph_replays(gpu):
    from turboquant_amd.eviction import select_evictions
    from turboquant_amd.exact import ExactPagedCache
    seqs = Sequences([200, 200], 2, 64, torch.bfloat16)
    start = seqs.kv.clone()
    w, pos = weights_of(2, 2, 200, 0).to(gpu), in_order(2, 2, 200).to(gpu)
    lens, cache = seqs.seq_lens.clone(), ExactPagedCache.from_engine(seqs.kv)

    def step():
        e = select_evictions(w, pos, lens, 64, recent=16, out=None)
        cache.move_tokens(e, seqs.table)
        return e
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed, now in ((1, [200, 150]), (2, [64, 10]), (3, [65, 199])):
        seqs.kv.copy_(start)
        w.copy_(weights_of(2, 2, 200, seed))
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        moved = seqs.kv.clone()
        seqs.kv.copy_(start)
        want = step()
        for a, b in zip(got[:6], want[:6]):
            assert torch.equal(a, b)
        assert torch.equal(moved.view(torch.int16), seqs.kv.view(torch.int16))


def test_refusals(gpu):
    from turboquant_amd.eviction import select_evictions
    from turboquant_amd.exact import ExactPagedCache
    w, pos, lens = torch.zeros(2, 2, 40, device=gpu), in_order(2, 2, 40).to(gpu), torch.tensor([40, 40], device=gpu)
    ok = lambda **kw: select_evictions(**{**dict(weights=w, positions=pos, seq_lens=lens, budget=20), **kw})
    e = ok()
    both = torch.zeros(2, 2, 80, device=gpu)
    for bad, error in ((dict(budget=0), ValueError), (dict(budget=2 ** 32 + 5), ValueError), (dict(sinks=-1), ValueError), (dict(recent=-1), ValueError), (dict(sinks=10, recent=11), ValueError),
                       (dict(weights=w.cpu()), RuntimeError), (dict(positions=pos.cpu()), RuntimeError), (dict(weights=w[0]), ValueError),
                       (dict(positions=pos[..., :39]), ValueError), (dict(weights=w.double()), TypeError), (dict(positions=pos.long()), TypeError),
                       (dict(seq_lens=lens[:1]), ValueError), (dict(seen=lens[:1]), ValueError), (dict(out=(w, pos[..., :39])), ValueError),
                       (dict(out=(w[:, :, :39], pos)), ValueError), (dict(out=(w[:1].expand(2, 2, 40), pos)), ValueError),
                       (dict(out=(both[..., 40:].clone().requires_grad_(), pos)), RuntimeError),
                       (dict(weights=both[..., :40], out=(both[..., 1:41], pos)), ValueError),
                       (dict(out=(pos.view(torch.float32), torch.zeros_like(pos))), ValueError),
                       (dict(out=(both[..., :40], both.view(torch.int32)[..., 20:60])), ValueError),
                       (dict(weights=w[..., :0], positions=pos[..., :0]), ValueError)):
        with pytest.raises(error):
            ok(**bad)
    seqs = Sequences([40, 40], 2, 64, torch.bfloat16)
    cache = ExactPagedCache.from_engine(seqs.kv)
    cache.move_tokens(e, seqs.table)
    for table in (seqs.table[:1], seqs.table.long(), seqs.table[0], seqs.table[:, :0], ):
        with pytest.raises(ValueError):
            cache.move_tokens(e, table)
    with pytest.raises(RuntimeError):
        cache.move_tokens(e, seqs.table.cpu())
    with pytest.raises(ValueError):
        ExactPagedCache.from_engine(seqs.kv[:, :, :, :1]).move_tokens(e, seqs.table)
    for bad in (e._replace(src=e.src[..., :1]), e._replace(dst=e.dst.long()), e._replace(count=e.count[:1]),
                e._replace(dst=e.dst[..., ::2], src=e.src[..., ::2])):
        with pytest.raises(ValueError):
            cache.move_tokens(bad, seqs.table)
    none = select_evictions(w[:0], pos[:0], lens[:0], 20)
    assert none.lens.shape == (0,)
    cache.move_tokens(none, seqs.table[:0])
