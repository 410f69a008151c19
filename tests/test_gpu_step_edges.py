"""A step's operators at their limits: offsets beyond 32 bits, the most heads, other streams, shared prefixes, and what they refuse."""

import math

import pytest
import torch

from tests.step_helpers import F8, PAGE, Step
from turboquant_amd.exact import ExactPagedCache
from turboquant_amd.fp8 import Fp8PagedCache
from turboquant_amd.rotary import inverse_frequencies, rotate_heads

pytestmark = pytest.mark.gpu

KINDS = {"bf16": (torch.bfloat16, torch.bfloat16), "fp8": ("fp8", torch.bfloat16)}


def moved(s, far, spread):
    """Step s with its blocks from number `far` on (spread None), or `spread` bytes apart, in a cache of its own."""
    size = s.q[0].element_size()
    shape = s.q[0].shape
    if spread is None:
        new = [torch.empty(far + s.blocks, *shape[1:], dtype=x.dtype, device=x.device) for x in s.q]
        for x, y in zip(new, s.q):
            x[far:].view(torch.uint8).copy_(y.view(torch.uint8))
        table = torch.where(s.table >= 0, s.table + far, s.table)
        scales = [torch.cat([torch.zeros(far, s.H, dtype=torch.uint8, device=x.device), x]) for x in s.scales] if size == 1 else []
    else:
        new = []
        for y in s.q:
            room = torch.empty(spread * (s.blocks - 1) + y[0].numel() * size, dtype=torch.uint8, device=y.device).view(y.dtype)
            x = room.as_strided(shape, (spread // size, *y.stride()[1:]))
            x.view(torch.uint8).copy_(y.view(torch.uint8))
            new.append(x)
        table, scales = s.table, s.scales if size == 1 else []
    return (Fp8PagedCache if size == 1 else ExactPagedCache)(*new, *scales), table


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("spread", [None, (1 << 32) + 256])
def test_blocks_beyond_32_bits(gpu, kind, spread):
    lens, runs = [70, 20], [40, 3]
    s = Step(lens, runs, 8, 128, *KINDS[kind], spare=0)
    q = s.query(16).to(gpu)
    block = 16 * 8 * 128 * s.q[0].element_size()
    cache, table = moved(s, (1 << 32) // block + 5, spread)
    for window, sinks in ((None, 0), (30, 2)):
        kw = dict(window=window, sinks=sinks)
        got = cache.attention(q, s.starts, table, s.seq_lens, **kw)
        assert torch.equal(got, s.cache().attention(q, s.starts, s.table, s.seq_lens, **kw))
        s.check(q.cpu(), got, 1 / math.sqrt(128), window, sinks)
        got = cache.decode_attention(q[:2], table, s.seq_lens, window=window or 1000, sinks=sinks)
        assert torch.equal(got, s.cache().decode_attention(q[:2], s.table, s.seq_lens, window=window or 1000, sinks=sinks))
    if kind == "fp8":
        k, v = (torch.randn(43, 8, 128, device=gpu, dtype=torch.bfloat16) for _ in range(2))
        read = []
        for c, t in ((cache, table), (s.cache(), s.table)):
            c.write(k, v, s.starts, t, s.seq_lens)
            read.append(c.read(s.starts, t, s.seq_lens, rows=43))
        assert all(torch.equal(a, b) for a, b in zip(*read))


def test_rows_beyond_32_bits(gpu):
    """More than 2^31 elements of queries, of keys to write and to read, of heads to rotate: the last rows' results are those of the rows alone."""
    H, d, n = 8, 128, 20
    rows = (1 << 31) // (H * d) + 1000
    B = 64
    run = (rows + B - 1) // B
    rows = run * B
    pages = (run + PAGE - 1) // PAGE
    x = torch.empty(rows, H, d, dtype=torch.bfloat16, device=gpu)
    for part in x.split(1 << 17):
        part.normal_()
    table = torch.arange(B * pages, dtype=torch.int32, device=gpu).view(B, pages)
    lens = torch.full((B,), run, dtype=torch.int32, device=gpu)
    starts = torch.arange(B + 1, dtype=torch.int32, device=gpu) * run
    cache = Fp8PagedCache.allocate(B * pages, H, d, gpu)
    cache.write(x, x, starts, table, lens)
    alone = Fp8PagedCache.allocate(pages, H, d, gpu)
    one = torch.tensor([0, run], dtype=torch.int32, device=gpu)
    alone.write(x[-run:].clone(), x[-run:].clone(), one, table[:1], lens[:1])
    assert all(torch.equal(a[-pages:].view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache.operands(), alone.operands()))
    k, v = cache.read(starts, table, lens, rows=rows)
    few = alone.read(one, table[:1], lens[:1], rows=run)
    assert torch.equal(k[-run:], few[0]) and torch.equal(v[-run:], few[1])
    del k, v
    # 16 query heads on each of 8 would be 8 times the memory: the rows' own heads as queries, within a window so that it stays quick
    got = cache.attention(x, starts, table, lens, window=40, max_rows=run)
    want = alone.attention(x[-run:].clone(), one, table[:1], lens[:1], window=40, max_rows=run, n_split=1)
    assert ((got[-run:].float() - want.float()).abs() <= 2.0 ** -7 * (want.float().abs() + 1)).all()
    del got, want
    positions = torch.arange(rows, device=gpu)
    f = inverse_frequencies(d, device=gpu)
    q, k = rotate_heads(x, x[:, :1], positions, f)
    q2, k2 = rotate_heads(x[-n:].clone(), x[-n:, :1].clone(), positions[-n:].clone(), f)
    assert torch.equal(q[-n:], q2) and torch.equal(k[-n:], k2)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("G,runs", [(1024, [1, 1]), (1024, [2, 3]), (33, [1, 4])])
def test_many_heads_on_one(gpu, kind, G, runs):
    s = Step([130, 9], runs, 1, 64, *KINDS[kind])
    q = s.query(G)
    s.check(q, s.cache().attention(q.to(gpu), s.starts, s.table, s.seq_lens, window=50, sinks=1), 1 / 8, 50, 1)
    with pytest.raises(ValueError):
        s.cache().attention(torch.zeros(s.rows, 1025, 64, dtype=s.dtype, device=gpu), s.starts, s.table, s.seq_lens, window=50)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("runs", [[1, 1, 1], [9, 30, 2]])
def test_a_prefix_that_sequences_share(gpu, kind, runs):
    """The same blocks in several tables: read by all of them."""
    s = Step([100, 100, 100], runs, 2, 64, *KINDS[kind])
    table = s.table.clone()
    table[1, :4], table[2] = table[0, :4], table[0]
    s.table, s.table_cpu = table, table.cpu()
    q = s.query(4)
    s.check(q, s.cache().attention(q.to(gpu), s.starts, table, s.seq_lens), 1 / 8)


@pytest.mark.parametrize("kind", list(KINDS))
def test_other_streams(gpu, kind):
    """Two streams at once, each with tensors of its own; results as on the default one."""
    steps = [Step([600, 90], r, 2, 128, *KINDS[kind], seed=i) for i, r in enumerate(([1, 1], [50, 7]))]
    asked = [s.query(8).to(gpu) for s in steps]
    want = [s.cache().attention(q, s.starts, s.table, s.seq_lens) for s, q in zip(steps, asked)]
    streams = [torch.cuda.Stream() for _ in steps]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(steps[i].cache().attention(asked[i], steps[i].starts, steps[i].table, steps[i].seq_lens))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for gs, w in zip(got, want) for g in gs)


def test_lengths_on_the_host_and_in_64_bits(gpu):
    s = Step([70, 20], [5, 1], 2, 64, *KINDS["fp8"])
    q = s.query(4).to(gpu)
    want = s.cache().attention(q, s.starts, s.table, s.seq_lens)
    assert torch.equal(want, s.cache().attention(q, s.starts.long().cpu(), s.table, s.seq_lens.long().cpu()))
    assert torch.equal(want, s.cache().attention(q, s.starts.long(), s.table.repeat(1, 2)[:, : s.width], s.seq_lens.double().long()))


def test_attention_refuses(gpu):
    for kind in KINDS:
        s = Step([70, 20], [5, 1], 2, 64, *KINDS[kind])
        c, q = s.cache(), s.query(4).to(gpu)
        call = lambda q=q, starts=s.starts, table=s.table, lens=s.seq_lens, **kw: c.attention(q, starts, table, lens, **kw)
        call()
        held = c.key_cache.view(torch.uint8) if kind == "fp8" else c.key_cache
        for bad in (dict(window=0), dict(window=-3), dict(window=1 << 31), dict(sinks=2), dict(window=5, sinks=-1), dict(n_split=-1), dict(n_split=1025),
                    dict(max_len=-1), dict(max_rows=-1), dict(table=s.table.long()), dict(table=s.table[:1]), dict(table=s.table[:, :0]), dict(lens=s.seq_lens[:1]),
                    dict(starts=s.starts[None]), dict(starts=s.starts[:0]), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q[0]), dict(out=q), dict(out=q[:3].clone()),
                    dict(out=torch.empty_like(q).float()), dict(out=torch.empty(6, 4, 128, dtype=q.dtype, device=gpu)[..., ::2]),
                    dict(out=held.flatten()[: q.numel() * 2].view(torch.bfloat16)[: q.numel()].view_as(q)) if kind == "fp8" else dict(out=c.key_cache.flatten()[: q.numel()].view_as(q)),
                    dict(workspace=torch.empty(4, device=gpu)), dict(workspace=torch.empty(1 << 20, device=gpu)[1:])):
            with pytest.raises(ValueError):
                call(**bad)
        for bad in (dict(q=q.float()), dict(q=q.double())) + (() if kind == "fp8" else (dict(q=q.half()),)):
            with pytest.raises(TypeError):
                call(**bad)
        with pytest.raises(RuntimeError):
            call(q=q.cpu())
        with pytest.raises(RuntimeError):
            call(q=q.clone().requires_grad_())
        with torch.no_grad():
            assert torch.equal(call(q=q.clone().requires_grad_()), call())
    wide = ExactPagedCache(*(torch.zeros(4, 16, 2, 320, dtype=torch.bfloat16, device=gpu) for _ in range(2)))
    with pytest.raises(ValueError):
        wide.attention(torch.zeros(6, 4, 320, dtype=torch.bfloat16, device=gpu), s.starts, s.table, s.seq_lens)
    single = ExactPagedCache(*(torch.zeros(4, 16, 2, 64, device=gpu) for _ in range(2)))
    with pytest.raises(TypeError):
        single.attention(torch.zeros(6, 4, 64, device=gpu), s.starts, s.table, s.seq_lens)
    exact = Step([70, 20], [1, 1], 2, 64, *KINDS["bf16"])
    with pytest.raises(ValueError):
        exact.cache().decode_attention(exact.query(4).to(gpu), exact.table, exact.seq_lens, window=8, weights=torch.zeros(2, 2, 128, device=gpu))


def test_the_cache_refuses(gpu):
    c = Fp8PagedCache.allocate(4, 2, 64, gpu)
    k = torch.zeros(6, 2, 64, dtype=torch.bfloat16, device=gpu)
    starts, table, lens = (torch.tensor(x, dtype=torch.int32, device=gpu) for x in ([0, 5, 6], [[0, 1], [2, 3]], [20, 3]))
    c.write(k, k, starts, table, lens)
    for a in ((k[:5], k, starts, table, lens), (k[..., :32], k[..., :32], starts, table, lens), (k, k, starts[:2], table, lens), (k, k, starts, table[0], lens),
              (k, k, starts, table.long(), lens), (k, k, starts, table, lens[:1]),
              (c.key_cache.view(torch.bfloat16).flatten()[: k.numel()].view_as(k), k, starts, table, lens)):
        with pytest.raises(ValueError):
            c.write(*a)
    with pytest.raises(TypeError):
        c.write(k, k.half(), starts, table, lens)
    with pytest.raises(RuntimeError):
        c.write(k.float().requires_grad_(), k.float(), starts, table, lens)
    with pytest.raises(RuntimeError):
        c.write(k.cpu(), k, starts, table, lens)
    for bad in (dict(), dict(rows=-1), dict(out=(k, k)), dict(out=(k, k.clone()), rows=5), dict(out=(k.half(), k.clone())), dict(out=(k[..., ::2], k))):
        with pytest.raises(ValueError):
            c.read(starts, table, lens, **bad)
    q8 = lambda *shape: torch.zeros(*shape, dtype=torch.uint8, device=gpu).view(F8)
    sc = torch.zeros(4, 2, dtype=torch.uint8, device=gpu)
    for blocks, scales in (((q8(4, 16, 2, 96),) * 2, (sc, sc)), ((q8(4, 16, 2, 64), q8(4, 16, 3, 64)), (sc, sc)), ((q8(4, 8, 2, 64),) * 2, (sc, sc)),
                           ((q8(4, 16, 2, 64),) * 2, (sc[:3], sc)), ((q8(4, 16, 2, 64),) * 2, (sc.t(), sc)), ((q8(4, 16, 2, 72)[..., :64],) * 2, (sc, sc))):
        with pytest.raises(ValueError):
            Fp8PagedCache(*blocks, *scales)
    for blocks, scales in (((q8(4, 16, 2, 64).view(torch.uint8),) * 2, (sc, sc)), ((q8(4, 16, 2, 64),) * 2, (sc.int(), sc))):
        with pytest.raises(TypeError):
            Fp8PagedCache(*blocks, *scales)
    folded = Fp8PagedCache(q8(1, 16, 2, 64).expand(4, -1, -1, -1), q8(1, 16, 2, 64).expand(4, -1, -1, -1), sc, sc.clone())
    with pytest.raises(ValueError):
        folded.write(k, k, starts, table, lens)
    folded.read(starts, table, lens, rows=6)                  # (to read, blocks may be one)


def test_rotation_refuses(gpu):
    q, k = torch.randn(6, 4, 64, device=gpu), torch.randn(6, 2, 64, device=gpu)
    pos, f = torch.arange(6, device=gpu), inverse_frequencies(64, device=gpu)
    w = torch.ones(64, device=gpu)
    rotate_heads(q, k, pos, f, w, w)
    for a in ((q, k[:5], pos, f), (q, k[..., :32], pos, f), (q[0], k[0], pos, f), (q, k, pos[:5], f), (q, k, pos.float(), f), (q, k, pos, f.float()), (q, k, pos, f[None]),
              (q, k, pos, inverse_frequencies(128, device=gpu)), (q, k, pos, f[:30]), (q[..., :60], k[..., :60], pos, f[:28]), (q, k, pos, f, w[:32]), (q, k, pos, f, w.half()),
              (q, k, pos, f, None, w.cpu())):
        with pytest.raises(ValueError):
            rotate_heads(*a)
    with pytest.raises(TypeError):
        rotate_heads(q, k.half(), pos, f)
    with pytest.raises(RuntimeError):
        rotate_heads(q, k, pos.cpu(), f)
    with pytest.raises(RuntimeError):
        rotate_heads(q, k, pos, f, w.clone().requires_grad_())
    for out in ((q, q), (q, torch.empty_like(q)), (q[:5], k), (q.clone(), k.double()), (k, k), (torch.empty(1, 4, 64, device=gpu).expand(6, -1, -1), k.clone())):
        with pytest.raises(ValueError):
            rotate_heads(q, k, pos, f, out=out)


@pytest.mark.parametrize("kind", ["fp8", "fp8 fp16"])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("runs", [[1, 1], [5, 2], [60, 20]])
def test_scales_of_blocks_that_hold_nothing(gpu, kind, d, runs):
    """A cache that was never cleared: bytes of NaN and scales of 2^128 wherever no sequence's token is, block 0 among them; entries outside the cache."""
    s = Step([100, 90], runs, 2, d, "fp8", torch.float16 if kind == "fp8 fp16" else torch.bfloat16, spare=40, seed=1)
    used = s.table_cpu[s.table_cpu >= 0].long()
    assert 0 not in used
    empty = torch.ones(s.blocks, dtype=torch.bool)
    empty[used] = False
    for scales in s.scales:
        scales[empty.to(gpu)] = 255
    for bad in (-1, s.blocks, 2 ** 31 - 1):
        s.table_cpu[0, 2], s.table_cpu[1, 0] = bad, bad
        s.table = s.table_cpu.to(gpu)
        q = s.query(8)
        for window, sinks in ((None, 0), (40, 3)):
            s.check(q, s.cache().attention(q.to(gpu), s.starts, s.table, s.seq_lens, window=window, sinks=sinks), 1 / math.sqrt(d), window, sinks)


def test_frequencies_that_want_gradients(gpu):
    q, k = torch.randn(3, 2, 64, device=gpu), torch.randn(3, 1, 64, device=gpu)
    f = inverse_frequencies(64, device=gpu).requires_grad_()
    with pytest.raises(RuntimeError):
        rotate_heads(q, k, torch.arange(3, device=gpu), f)


def test_keys_and_values_in_one_place(gpu):
    """Written to, a cache's four tensors are memory of their own; values in the gaps between keys are."""
    H, d, n = 2, 64, 4
    bytes_ = lambda *shape: torch.zeros(*shape, dtype=torch.uint8, device=gpu)
    scales = [bytes_(n, H) for _ in range(2)]
    k, v = (torch.randn(20, H, d, device=gpu, generator=torch.Generator(gpu).manual_seed(i)) for i in range(2))
    step = [torch.tensor(x, dtype=torch.int32, device=gpu) for x in ([0, 20], [[2, 1]], [20])]
    one = bytes_(n, PAGE, H, d).view(F8)
    for bad in ((one, one, *scales), (one[:-1], one[1:], *(s[:-1] for s in scales)), (one, bytes_(n, PAGE, H, d).view(F8), scales[0], scales[0]),
                (one, bytes_(n, PAGE, H, d).view(F8), scales[0], one.view(torch.uint8).flatten()[: n * H].view(n, H))):
        cache = Fp8PagedCache(*bad)
        with pytest.raises(ValueError, match="overlaps itself"):
            cache.write(k, v, *step)
        cache.read(*step, rows=20)
    apart = Fp8PagedCache.allocate(n, H, d, gpu)
    apart.write(k, v, *step)
    want = apart.read(*step, rows=20)
    blocks = bytes_(n, 2, PAGE, H, d).view(F8)
    sides = bytes_(n, PAGE, H, 2 * d).view(F8)
    rows = bytes_(n, PAGE, 2, H, d).view(F8)
    for a, b in ((blocks[:, 0], blocks[:, 1]), (blocks[:, 1], blocks[:, 0]), (sides[..., :d], sides[..., d:]), (rows[:, :, 0], rows[:, :, 1])):
        cache = Fp8PagedCache(a, b, bytes_(n, H), bytes_(n, H))
        cache.write(k, v, *step)
        assert all(torch.equal(x, y) for x, y in zip(cache.read(*step, rows=20), want))


def test_rotation_over_what_it_reads(gpu):
    room = torch.zeros(4, 64, dtype=torch.float64, device=gpu)
    q, k, f = torch.randn(4, 1, 64, device=gpu), torch.randn(4, 1, 64, device=gpu), room[0, :32]
    with pytest.raises(ValueError, match="inv_freq"):
        rotate_heads(q, k, torch.arange(4, device=gpu), f, out=(room.view(torch.float32)[:, None, :64], k.clone()))


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("G", [1, 4, 16, 64])
@pytest.mark.parametrize("runs", [[1], [3], [1, 0, 2], [16], [33, 1]])
@pytest.mark.parametrize("extra", [1, 2, 40])
def test_rows_of_no_sequence_behind_full_units(gpu, kind, G, runs, extra):
    """The units of a step may be as many as there can be: rows of no sequence are zeros all the same, or as they were."""
    s = Step([300 + 7 * i for i in range(len(runs))], runs, 2, 64, *KINDS[kind], extra=extra)
    q = s.query(2 * G).to(gpu)
    for kw in (dict(), dict(n_split=1), dict(n_split=5), dict(max_len=16), dict(window=50, sinks=2)):
        got = s.cache().attention(q, s.starts, s.table, s.seq_lens, **kw)
        assert (got[sum(runs):] == 0).all()
        out = torch.full_like(got, 3.0)
        s.cache().attention(q, s.starts, s.table, s.seq_lens, out=out, **kw)
        assert (out[sum(runs):] == 3).all() and torch.equal(out[: sum(runs)], got[: sum(runs)])
    late = s.starts + extra                                  # rows in front of the first sequence
    moved = torch.cat([q[sum(runs):], q[: sum(runs)]])
    got2 = s.cache().attention(moved, late, s.table, s.seq_lens, window=50, sinks=2)
    assert (got2[:extra] == 0).all() and torch.equal(got2[extra:], got[: sum(runs)])
