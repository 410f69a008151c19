"""Decode attention over the engine's paged exact cache against 64 bits: types, head layouts, lengths, strides, block tables, streams, graphs."""

import pytest
import torch

from tests.exact_helpers import DTYPES, PAGE, Sequences, check_decode

pytestmark = pytest.mark.gpu


def decode(seqs, q, weights=None, **kw):
    from turboquant_amd.exact import ExactPagedCache
    return ExactPagedCache.from_engine(seqs.kv).decode_attention(q.to(seqs.device), seqs.table, seqs.seq_lens, weights=weights, **kw)


def start_weights(seqs, L, seed=7):
    w = torch.rand(len(seqs.lens), seqs.H, L, generator=torch.Generator().manual_seed(seed))
    return w, w.to(seqs.device)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("d", range(64, 769, 64))
def test_every_head_size(gpu, d, dtype):
    seqs = Sequences([0, 1, 15, 16, 17, 33, 150], 2, d, DTYPES[dtype], seed=d)
    q = seqs.query(7, 6, d)
    before, w = start_weights(seqs, 150)
    out = decode(seqs, q, w)
    assert out.dtype == seqs.dtype
    check_decode(seqs, q, out, d ** -0.5, before, w)
    assert not out[0].any()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("heads,H", [(1, 1), (2, 2), (3, 1), (10, 2), (15, 1), (16, 1), (17, 1), (48, 3), (72, 3), (128, 1), (200, 1)])
def test_heads_per_kv_head(gpu, heads, H, dtype):
    seqs = Sequences([5, 129, 700], H, 128, DTYPES[dtype], seed=heads)
    q = seqs.query(3, heads, 128)
    before, w = start_weights(seqs, 700)
    check_decode(seqs, q, decode(seqs, q, w), 128 ** -0.5, before, w)


# a bound on the lengths with which more than sixteen heads share their reads, however short the sequences are
SHARED = 1 << 21


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", range(64, 577, 64))
def test_heads_that_share_their_reads(gpu, d, dtype):
    seqs = Sequences([0, 1, 15, 16, 17, 33, 150], 2, d, DTYPES[dtype], seed=d)
    for heads in (34, 100):
        q = seqs.query(7, heads, d)
        before, w = start_weights(seqs, 150)
        check_decode(seqs, q, decode(seqs, q, w, max_len=SHARED), d ** -0.5, before, w)
    seqs = Sequences([2500, 31], 1, d, DTYPES[dtype], seed=d)
    q = seqs.query(2, 70, d)
    for splits in (1, 1024):                                       # one part, two
        before, w = start_weights(seqs, 2500)
        check_decode(seqs, q, decode(seqs, q, w, max_len=SHARED, n_split=splits), d ** -0.5, before, w)


@pytest.mark.parametrize("layout", ["engine", "heads", "padded"])
@pytest.mark.parametrize("dtype,d,heads", [("bf16", 128, 96), ("fp16", 256, 51), ("bf16", 512, 60), ("fp16", 576, 384)])
def test_heads_that_share_their_reads_layouts_and_blocks(gpu, dtype, d, heads, layout):
    seqs = Sequences([77, 300, 64], 3, d, DTYPES[dtype], layout=layout)
    q = seqs.query(3, heads, d)
    keep = [torch.ones(n, dtype=torch.bool) for n in seqs.lens]
    for b, page, entry in ((1, 3, -1), (1, 18, seqs.blocks), (2, 0, 2 ** 31 - 1), (2, 1, -2 ** 31), (2, 2, seqs.blocks), (2, 3, -7)):
        seqs.table[b, page] = entry
        keep[b][page * PAGE: (page + 1) * PAGE] = False
    before, w = start_weights(seqs, 300)
    out = decode(seqs, q, w, scale=0.07, max_len=SHARED)
    check_decode(seqs, q, out, 0.07, before, w, keep=keep)
    assert not out[2].any()


def test_many_heads_over_a_cache_of_some_length(gpu):
    """Sizes at which the heads share their reads without being told, several parts to a sequence."""
    seqs = Sequences([1400, 2, 900], 1, 576, torch.bfloat16)
    q = seqs.query(3, 128, 576)
    before, w = start_weights(seqs, 1400)
    check_decode(seqs, q, decode(seqs, q, w), 576 ** -0.5, before, w)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n", [1, 2, 16, 31, 32, 33, 127, 128, 129, 511, 513, 1024, 1025, 4097])
def test_lengths_and_splits(gpu, n, dtype):
    seqs = Sequences([n, max(0, n - 16)], 1, 64, DTYPES[dtype], seed=n)
    q = seqs.query(2, 4, 64)
    for splits in (None, 1, 2, 3, 7, 64, 1024):
        before, w = start_weights(seqs, n)
        check_decode(seqs, q, decode(seqs, q, w, n_split=splits), 0.125, before, w)


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("fp16", 256), ("fp32", 64), ("bf16", 576)])
@pytest.mark.parametrize("layout", ["engine", "heads", "padded"])
def test_layouts(gpu, layout, dtype, d):
    seqs = Sequences([77, 300], 3, d, DTYPES[dtype], layout=layout)
    q = seqs.query(2, 9, d)
    before, w = start_weights(seqs, 300)
    check_decode(seqs, q, decode(seqs, q, w, scale=0.07), 0.07, before, w)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_blocks_outside_the_cache_have_no_weight(gpu, dtype):
    seqs = Sequences([200, 64, 90], 2, 64, DTYPES[dtype])
    q = seqs.query(3, 4, 64)
    keep = [torch.ones(n, dtype=torch.bool) for n in seqs.lens]
    for b, page, entry in ((0, 3, -1), (0, 12, seqs.blocks), (1, 0, 2 ** 31 - 1), (1, 1, -2 ** 31), (1, 2, seqs.blocks), (1, 3, -7)):
        seqs.table[b, page] = entry
        keep[b][page * PAGE: (page + 1) * PAGE] = False
    before, w = start_weights(seqs, 200)
    out = decode(seqs, q, w)
    check_decode(seqs, q, out, 0.125, before, w, keep=keep)
    assert not out[1].any()


def test_one_table_for_all_and_a_table_shorter_than_the_lengths(gpu):
    seqs = Sequences([100, 100], 2, 128, torch.bfloat16)
    seqs.k64[1], seqs.v64[1] = seqs.k64[0], seqs.v64[0]
    q = seqs.query(2, 8, 128)
    seqs.table = seqs.table[0]
    seqs.seq_lens = torch.tensor([100, 37], dtype=torch.int32, device=seqs.device)
    before, w = start_weights(seqs, 100)
    check_decode(seqs, q, decode(seqs, q, w), 128 ** -0.5, before, w, lens=[100, 37])
    seqs.table = seqs.table[:4]                                     # 64 tokens
    before, w = start_weights(seqs, 100)
    check_decode(seqs, q, decode(seqs, q, w), 128 ** -0.5, before, w, lens=[64, 37])
    seqs.seq_lens = torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32, device=seqs.device)
    before, w = start_weights(seqs, 100)
    check_decode(seqs, q, decode(seqs, q, w), 128 ** -0.5, before, w, lens=[64, 0])


@pytest.mark.parametrize("max_len", [0, 1, 40, 5000])
def test_a_bound_on_the_lengths_is_only_a_plan(gpu, max_len):
    seqs = Sequences([3000, 5, 700], 2, 64, torch.float16)
    q = seqs.query(3, 4, 64)
    before, w = start_weights(seqs, 3000)
    check_decode(seqs, q, decode(seqs, q, w, max_len=max_len), 0.125, before, w)


def test_weights_with_strides_and_fewer_places_than_tokens(gpu):
    seqs = Sequences([300, 20, 257], 2, 128, torch.bfloat16)
    q = seqs.query(3, 8, 128)
    for L in (1, 16, 200, 257, 300, 400):
        whole = torch.rand(2, 3, L + 5, generator=torch.Generator().manual_seed(3))
        held = whole.to(seqs.device)
        w = held.transpose(0, 1)[:, :, :L]
        check_decode(seqs, q, decode(seqs, q, w), 128 ** -0.5, whole.transpose(0, 1)[:, :, :L], w)
        assert torch.equal(held[:, :, L:].cpu(), whole[:, :, L:])


def test_weights_do_not_change_the_output_and_repeat(gpu):
    seqs = Sequences([1000, 333, 4000], 4, 128, torch.bfloat16)
    q = seqs.query(3, 32, 128)
    plain = decode(seqs, q)
    w1, w2 = (torch.zeros(3, 4, 4000, device=seqs.device) for _ in range(2))
    assert torch.equal(plain, decode(seqs, q, w1)) and torch.equal(plain, decode(seqs, q, w2)) and torch.equal(w1, w2)


def test_large_scores_and_a_token_that_takes_it_all(gpu):
    """Scores hundreds apart: all weight on one token, none lost to the others' rounding; and equal scores: the mean."""
    for dt in DTYPES.values():
        seqs = Sequences([600], 1, 64, dt)
        q = seqs.query(1, 2, 64)
        check_decode(seqs, q, decode(seqs, q, scale=20.0), 20.0)
        check_decode(seqs, q, decode(seqs, q, scale=0.0), 0.0)
        check_decode(seqs, q, decode(seqs, q, scale=-0.3), -0.3)


def test_long_context_of_small_weights_in_fp16(gpu):
    """One token far above 40,000 others, whose weights fp16 could not hold by themselves."""
    n = 40000
    seqs = Sequences([n], 1, 64, torch.float16)
    k = torch.zeros(n, 1, 64, dtype=torch.float64)
    k[0, 0, 0] = 18.0 * 0.6931471805599453
    k = k.to(torch.float16).double()
    v = torch.ones(n, 1, 64, dtype=torch.float64)
    v[0] = -1.0
    at = torch.arange(n)
    for i, x in enumerate((k, v)):
        seqs.kv[i][seqs.table[0, at // PAGE].long().cpu(), at % PAGE] = x.to(torch.float16).to(seqs.device)
    seqs.k64, seqs.v64 = [k], [v]
    q = torch.zeros(1, 1, 64, dtype=torch.float16)
    q[0, 0, 0] = 1.0
    check_decode(seqs, q, decode(seqs, q, scale=1.0), 1.0)


def test_nan_and_infinity_where_tokens_are(gpu):
    """A NaN of a key reaches its own sequence and KV head, that of a value its channel; the others are as without."""
    seqs = Sequences([70, 70], 2, 64, torch.bfloat16)
    q = seqs.query(2, 4, 64)
    clean = decode(seqs, q)
    at = seqs.table[0, 2].long(), 3
    seqs.kv[0][at[0], at[1], 1, 5] = float("nan")
    out = decode(seqs, q)
    assert torch.isnan(out[0, 2:]).all() and torch.equal(out[0, :2], clean[0, :2]) and torch.equal(out[1], clean[1])
    seqs.kv[0][at[0], at[1], 1, 5] = 0.5
    clean = decode(seqs, q)
    seqs.kv[1][at[0], at[1], 0, 9] = float("inf")
    out = decode(seqs, q)
    assert torch.isinf(out[0, :2, 9]).all()
    out[0, :2, 9] = clean[0, :2, 9]
    assert torch.equal(out, clean)


def test_offsets_beyond_32_bits(gpu):
    """Blocks whose elements lie past 2^32 bytes and past 2^31 elements."""
    from turboquant_amd.exact import ExactPagedCache
    small = Sequences([100, 90], 8, 128, torch.bfloat16)
    blocks = (1 << 31) // (PAGE * 8 * 128) + 200
    k, v = (torch.empty(blocks, PAGE, 8, 128, dtype=torch.bfloat16, device=small.device) for _ in range(2))
    far = blocks - small.blocks
    k[far:], v[far:] = small.kv[0], small.kv[1]
    table = torch.where(small.table >= 0, small.table + far, small.table)
    q = small.query(2, 16, 128)
    before, w = start_weights(small, 100)
    out = ExactPagedCache(k, v).decode_attention(q.to(small.device), table, small.seq_lens, weights=w)
    check_decode(small, q, out, 128 ** -0.5, before, w)


def test_out_workspace_and_query_strides(gpu):
    from turboquant_amd.exact import ExactPagedCache
    seqs = Sequences([500, 40], 2, 128, torch.bfloat16)
    cache = ExactPagedCache.from_engine(seqs.kv)
    q = seqs.query(2, 8, 128)
    wide = torch.zeros(2, 8, 129, dtype=torch.bfloat16, device=seqs.device)
    wide[:, :, 1:] = q.to(seqs.device)
    out = torch.empty(2, 8, 128, dtype=torch.bfloat16, device=seqs.device)
    ws = cache.workspace(2, 8, 500, weight_len=500)
    before, w = start_weights(seqs, 500)
    got = cache.decode_attention(wide[:, :, 1:], seqs.table, seqs.seq_lens, weights=w, out=out, workspace=ws, max_len=500)
    assert got is out
    check_decode(seqs, q, out, 128 ** -0.5, before, w)
    assert cache.decode_attention(q[:0].to(seqs.device), seqs.table[:0], seqs.seq_lens[:0]).shape == (0, 8, 128)
    with pytest.raises(ValueError):
        cache.decode_attention(q.to(seqs.device), seqs.table, seqs.seq_lens, workspace=ws[:16])


def test_two_streams_at_once(gpu):
    a, b = Sequences([3000, 100], 2, 128, torch.bfloat16, seed=1), Sequences([50, 2500], 2, 128, torch.bfloat16, seed=2)
    qa, qb = a.query(2, 8, 128), b.query(2, 8, 128, seed=5)
    qa_d, qb_d = qa.to(gpu), qb.to(gpu)
    outs = []
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for st, s, q in zip(streams, (a, b), (qa_d, qb_d)):
            with torch.cuda.stream(st):
                outs.append(decode(s, q))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        check_decode((a, b)[i % 2], (qa, qb)[i % 2], o, 128 ** -0.5)


def test_graph_replays_with_lengths_that_grow(gpu):
    """Captured once; lengths and weights live on the device, eager calls run between the replays."""
    from turboquant_amd.exact import ExactPagedCache
    seqs = Sequences([1200, 600], 2, 128, torch.bfloat16)
    cache = ExactPagedCache.from_engine(seqs.kv)
    q = seqs.query(2, 8, 128)
    q_d, lens = q.to(gpu), torch.tensor([1000, 100], dtype=torch.int32, device=gpu)
    w = torch.zeros(2, 2, 1200, device=gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.decode_attention(q_d, seqs.table, lens, weights=w, max_len=1200)
    torch.cuda.current_stream().wait_stream(side)
    w.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.decode_attention(q_d, seqs.table, lens, weights=w, max_len=1200)
    before = torch.zeros(2, 2, 1200)
    for step in range(4):
        now = [1000 + 50 * step, 100 + 160 * step]
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        check_decode(seqs, q, out, 128 ** -0.5, before, w, lens=now)
        before = w.cpu().clone()
        eager = cache.decode_attention(q_d, seqs.table, lens, max_len=1200)
        assert torch.equal(eager, out)


def test_refusals(gpu):
    from turboquant_amd.exact import ExactPagedCache
    seqs = Sequences([40, 40], 2, 64, torch.bfloat16)
    kv, q = seqs.kv, seqs.query(2, 4, 64).to(gpu)
    cache = ExactPagedCache(kv[0], kv[1])
    ok = lambda **kw: cache.decode_attention(**{**dict(query=q, block_table=seqs.table, seq_lens=seqs.seq_lens), **kw})
    ok()
    for bad, error in ((dict(query=q[:, :3]), ValueError), (dict(query=q.float()), TypeError), (dict(query=q[..., :32]), ValueError),
                       (dict(query=q[0]), ValueError), (dict(query=q.cpu()), RuntimeError), (dict(block_table=seqs.table.long()), ValueError),
                       (dict(block_table=seqs.table[:1]), ValueError), (dict(block_table=seqs.table.cpu()), RuntimeError),
                       (dict(block_table=seqs.table[:, :0]), ValueError), (dict(seq_lens=seqs.seq_lens[:1]), ValueError),
                       (dict(n_split=-1), ValueError), (dict(n_split=1025), ValueError), (dict(max_len=-1), ValueError),
                       (dict(out=q[:, :2]), ValueError), (dict(out=q.float()), ValueError), (dict(out=torch._neg_view(q.clone())), ValueError),
                       (dict(out=q.clone().requires_grad_()), RuntimeError),
                       (dict(weights=torch.zeros(2, 2, 40, device=gpu, dtype=torch.float64)), TypeError),
                       (dict(weights=torch.zeros(2, 3, 40, device=gpu)), ValueError), (dict(weights=torch.zeros(2, 2, 40)), RuntimeError),
                       (dict(weights=torch.zeros(2, 2, 80, device=gpu)[..., ::2]), ValueError),
                       (dict(weights=torch.zeros(2, 1, 40, device=gpu).expand(2, 2, 40)), ValueError),
                       (dict(weights=torch.zeros(2, 2, 40, device=gpu, requires_grad=True)), RuntimeError),
                       (dict(query=q.clone().requires_grad_()), RuntimeError)):
        with pytest.raises(error):
            ok(**bad)
    with torch.no_grad():
        ok(query=q.clone().requires_grad_())
    for k, v, error in ((kv[0], kv[1].float(), TypeError), (kv[0].cpu(), kv[1], RuntimeError), (kv[0][:, :8], kv[1][:, :8], ValueError),
                        (kv[0], kv[1][:1], ValueError), (kv[0][..., :32], kv[1][..., :32], ValueError),
                        (kv[0].double(), kv[1].double(), TypeError), (kv[0], kv[1].transpose(2, 3).contiguous().transpose(2, 3), ValueError)):
        with pytest.raises(error):
            ExactPagedCache(k, v)
    odd = torch.zeros(kv.numel() + 1, dtype=kv.dtype, device=gpu)[1:].view(kv.shape)
    with pytest.raises(ValueError):
        ExactPagedCache(odd[0], odd[1])
    with pytest.raises(ValueError):
        ExactPagedCache.from_engine(kv[0])
