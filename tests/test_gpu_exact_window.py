"""The weights of a prompt's window over the paged exact cache against 64 bits."""

import pytest
import torch

from tests.exact_helpers import DTYPES, PAGE, Sequences, check_weights, window64

pytestmark = pytest.mark.gpu


def cache_of(seqs):
    from turboquant_amd.exact import ExactPagedCache
    return ExactPagedCache.from_engine(seqs.kv)


def case(seqs, rows, heads, window, scale=None, L=None, keep=None, **kw):
    """One call: `rows` query rows of each sequence, weights that hold something already."""
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    q = seqs.query(starts[-1], heads, seqs.d, seed=5)
    L = max(1, *seqs.lens) if L is None else L
    before = torch.rand(len(seqs.lens), seqs.H, L, generator=torch.Generator().manual_seed(9))
    w = before.to(seqs.device)
    scale = seqs.d ** -0.5 if scale is None else scale
    got = cache_of(seqs).add_window_weights(q.to(seqs.device), torch.tensor(starts, dtype=torch.int32, device=seqs.device), seqs.table,
                                            seqs.seq_lens, w, window, scale=scale, **kw)
    assert got is w
    check_weights(w, before, *window64(seqs, q, starts, window, scale, keep))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("d", range(64, 769, 64))
def test_every_head_size(gpu, d, dtype):
    seqs = Sequences([0, 1, 15, 16, 17, 33, 150], 2, d, DTYPES[dtype], seed=d)
    case(seqs, [0, 1, 15, 10, 17, 1, 40], 6, 20)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("heads,H,window", [(1, 1, 1), (1, 1, 15), (4, 2, 16), (3, 1, 17), (8, 1, 33), (16, 1, 17), (7, 1, 40), (128, 1, 3), (20, 2, 64)])
def test_rows_from_one_to_hundreds(gpu, heads, H, window, dtype):
    seqs = Sequences([200, 70], H, 128, DTYPES[dtype], seed=heads)
    case(seqs, [100, 70], heads, window)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("d,heads,H,window", [(64, 24, 1, 40), (128, 24, 1, 33), (192, 7, 1, 100), (256, 16, 2, 64), (256, 5, 1, 77), (256, 1, 1, 300), (320, 40, 1, 16)])
def test_hundreds_of_rows_in_wide_workgroups(gpu, d, heads, H, window, dtype):
    """Windows that some sequences fill, one has a part of, and one a single row of; a negative scale; hidden tokens in most blocks."""
    seqs = Sequences([350, 90, 33, 1], H, d, DTYPES[dtype], seed=heads)
    case(seqs, [310, 90, 1, 1], heads, window)
    case(seqs, [350, 20, 33, 0], heads, window, scale=-0.2)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n", [1, 16, 31, 32, 33, 129, 1023, 1024, 1025, 2100, 5000])
def test_lengths(gpu, n, dtype):
    seqs = Sequences([n, max(0, n - 16)], 1, 64, DTYPES[dtype], seed=n)
    for max_len in (None, 0, 64, 100000):
        case(seqs, [min(n, 9), 0], 4, 8, max_len=max_len)


@pytest.mark.parametrize("layout", ["engine", "heads", "padded"])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_layouts(gpu, layout, dtype):
    seqs = Sequences([77, 300], 3, 128, DTYPES[dtype], layout=layout)
    case(seqs, [77, 300], 9, 12, scale=0.07)
    case(seqs, [77, 300], 9, 12, scale=-1.5)


def test_rows_that_differ_from_the_window_and_a_first_row_that_is_not_zero(gpu):
    """Rows in front of the first sequence's and behind the last's belong to nobody; a start outside the rows is cut."""
    seqs = Sequences([50, 60], 2, 64, torch.bfloat16)
    q = seqs.query(40, 4, 64, seed=5)
    for starts in ([3, 20, 31], [0, 0, 40], [-5, 10, 1000], [30, 10, 12]):
        w = torch.zeros(2, 2, 60, device=gpu)
        cache_of(seqs).add_window_weights(q.to(gpu), torch.tensor(starts, dtype=torch.int32, device=gpu), seqs.table, seqs.seq_lens, w, 16)
        check_weights(w, torch.zeros(2, 2, 60), *window64(seqs, q, starts, 16, 0.125))


def test_blocks_outside_the_cache_and_rows_that_see_nothing(gpu):
    seqs = Sequences([100, 40], 2, 64, torch.float16)
    keep = [torch.ones(n, dtype=torch.bool) for n in seqs.lens]
    for b, page, entry in ((0, 2, -3), (1, 0, seqs.blocks), (1, 1, -1)):
        seqs.table[b, page] = entry
        keep[b][page * PAGE: (page + 1) * PAGE] = False
    # sequence 1 has tokens 32 .. 39 left: of its newest 20 rows the first 12 see none
    case(seqs, [30, 20], 4, 20, keep=keep)


def test_fewer_places_than_tokens_and_strides(gpu):
    seqs = Sequences([300, 20], 2, 128, torch.bfloat16)
    for L in (1, 17, 299, 400):
        case(seqs, [300, 20], 8, 32, L=L)


def test_values_play_no_part_and_two_calls_are_the_same(gpu):
    seqs = Sequences([700, 90], 2, 128, torch.bfloat16)
    q, starts = seqs.query(60, 8, 128).to(gpu), torch.tensor([0, 30, 60], dtype=torch.int32, device=gpu)
    got = []
    for _ in range(2):
        w = torch.zeros(2, 2, 700, device=gpu)
        cache_of(seqs).add_window_weights(q, starts, seqs.table, seqs.seq_lens, w, 30)
        got.append(w)
        seqs.kv[1].fill_(float("nan"))
    assert torch.equal(*got)


def test_one_row_is_a_decode_step(gpu):
    """The last row's weights are those of decode attention with that query."""
    seqs = Sequences([333, 64], 2, 128, torch.bfloat16)
    q = seqs.query(2, 8, 128).to(gpu)
    a, b = (torch.zeros(2, 2, 333, device=gpu) for _ in range(2))
    cache = cache_of(seqs)
    cache.decode_attention(q, seqs.table, seqs.seq_lens, weights=a)
    cache.add_window_weights(q, torch.arange(3, dtype=torch.int32, device=gpu), seqs.table, seqs.seq_lens, b, 1)
    # two sums of the same scores in another order: 2 (n + 64) half steps of fp32 relative
    assert ((a - b).abs() <= 4 * 400 * 2.0 ** -24 * a).all()


def test_graph_replays(gpu):
    seqs = Sequences([500, 260], 2, 128, torch.bfloat16)
    q, starts = seqs.query(40, 8, 128), [0, 20, 40]
    q_d, s_d, lens = q.to(gpu), torch.tensor(starts, dtype=torch.int32, device=gpu), seqs.seq_lens.clone()
    cache, w = cache_of(seqs), torch.zeros(2, 2, 500, device=gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.add_window_weights(q_d, s_d, seqs.table, lens, w, 20)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.add_window_weights(q_d, s_d, seqs.table, lens, w, 20)
    for now in ([500, 260], [100, 17], [499, 0], [33, 200]):
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        w.zero_()
        graph.replay()
        torch.cuda.synchronize()
        add, err = window64(seqs, q, starts, 20, 128 ** -0.5, lens=now)
        check_weights(w[:, :, : add.shape[2]], torch.zeros(2, 2, add.shape[2]), add, err)
        eager = torch.zeros_like(w)
        cache.add_window_weights(q_d, s_d, seqs.table, lens, eager, 20)
        assert torch.equal(eager, w)


def test_refusals(gpu):
    seqs = Sequences([40, 40], 2, 64, torch.bfloat16)
    q, starts, w = seqs.query(20, 4, 64).to(gpu), torch.tensor([0, 10, 20], dtype=torch.int32, device=gpu), torch.zeros(2, 2, 40, device=gpu)
    cache = cache_of(seqs)
    ok = lambda **kw: cache.add_window_weights(**{**dict(query=q, query_start_loc=starts, block_table=seqs.table, seq_lens=seqs.seq_lens,
                                                         weights=w, window=8), **kw})
    ok()
    for bad, error in ((dict(window=0), ValueError), (dict(window=1025), ValueError), (dict(query=q[:, :3]), ValueError),
                       (dict(query=q.float()), TypeError), (dict(query=q.cpu()), RuntimeError), (dict(query_start_loc=starts[:2]), ValueError),
                       (dict(query_start_loc=starts[:0]), ValueError), (dict(query_start_loc=starts[None]), ValueError),
                       (dict(weights=w[:1]), ValueError), (dict(weights=w.double()), TypeError), (dict(max_len=-1), ValueError),
                       (dict(block_table=seqs.table.long()), ValueError), (dict(query=q.clone().requires_grad_()), RuntimeError)):
        with pytest.raises(error):
            ok(**bad)
    before = w.clone()
    assert ok(query=q[:0], query_start_loc=starts * 0) is w and torch.equal(w, before)
