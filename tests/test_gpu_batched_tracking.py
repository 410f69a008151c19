"""Tracked weights as an engine's batch changes: rows that take another sequence, rows in another order, steps of several kinds, lengths, refusals."""

import pytest
import torch

from tests.exact_helpers import evict64
from turboquant_amd.integration import batched
from turboquant_amd.integration import vllm as single
from turboquant_amd.integration.batched import evict_batched, install_batched_hooks, track_weights
from turboquant_amd.integration.harness import MinimalRunner

pytestmark = pytest.mark.gpu

SIZE = dict(n_layers=2, hidden=256, num_heads=8, num_kv_heads=2, head_dim=64, ffn=512, vocab=500, batch=3, max_seq_len=200)
G = 4                                       # query heads on a KV head: what one query gives in all


def runner(gpu, track=192, window=16, batch=3, **hooks):
    r = MinimalRunner(device=gpu, seed=5, **SIZE)
    install_batched_hooks(r, r.num_blocks, **hooks)
    if track:
        track_weights(r, batch, track, window=window)
    return r


@pytest.fixture(autouse=True)
def mode_back():
    before = single.get_mode()
    yield
    single.set_mode(before)


def states(r):
    return list(r._tq_layer_states.values())


def prompt(r, lens, seed=0):
    toks = torch.randint(0, SIZE["vocab"], (sum(lens),), generator=torch.Generator().manual_seed(seed)).to(r.device)
    return r.step(toks, r.metadata(lens))


def decode(r, *tokens):
    return r.decode_step(torch.tensor(tokens, device=r.device))


def given(r):
    """What all queries so far have given to each row's tokens, per layer (B, H)."""
    return [s.weights.sum(-1).cpu() for s in states(r)]


def per_row(*counts):
    return torch.tensor([float(c) * G for c in counts])[:, None].expand(len(counts), 2)


def everything(r):
    return [t.clone() for s in states(r) for t in (s.weights, s.positions)] + [c.clone() for c in r.kv_caches] + [
        s.pool.data.clone() for s in states(r) if s.pool is not None]


def same(a, b):
    return all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))


# ---- steps ------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("mode", ["capture_only", "hybrid", "full_tq"])
def test_an_exact_layer_counts_every_step_in_every_mode(gpu, mode):
    r = runner(gpu, exact_layers=2, mode=mode)
    prompt(r, [50, 12, 90])
    for step in range(3):
        decode(r, step, 9, 4)
    for got in given(r):
        assert torch.allclose(got, per_row(19, 15, 19), rtol=1e-4)


def test_capture_only_and_hybrid_sum_the_same(gpu):
    a, b = (runner(gpu, exact_layers=2, mode=mode) for mode in ("capture_only", "hybrid"))
    for r, mode in ((a, "capture_only"), (b, "hybrid")):
        single.set_mode(mode)
        prompt(r, [50, 12, 90])
        decode(r, 1, 9, 4)
    for s, t in zip(states(a)[:1], states(b)[:1]):           # (the first layer: what it is given does not depend on the mode)
        assert torch.allclose(s.weights, t.weights, rtol=1e-5, atol=1e-7)


@pytest.mark.parametrize("exact", [0, 2])
def test_what_a_sequence_is_given_does_not_depend_on_the_others_in_its_step(gpu, exact):
    """A decoding sequence beside another's prompt: its token counts as in a step of its own - in exact layers, not in compressed ones."""
    r = runner(gpu, exact_layers=exact, mode="hybrid")
    prompt(r, [50, 12, 0])
    before = [s.weights.clone() for s in states(r)]
    prompt(r, [1, 1, 30], seed=1)
    decoded = 1 if exact else 0
    for got, s, w in zip(given(r), states(r), before):
        assert torch.allclose(got, per_row(16 + decoded, 12 + decoded, 16), rtol=1e-4)
        if not exact:
            assert torch.equal(s.weights[:2], w[:2])
    decode(r, 1, 2, 3)
    for got in given(r):
        assert torch.allclose(got, per_row(16 + 2 * decoded, 12 + 2 * decoded, 16 + decoded), rtol=1e-4)


# ---- rows -------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("exact", [0, 2])
def test_a_row_that_takes_another_sequence_starts_anew(gpu, exact):
    r, fresh = (runner(gpu, exact_layers=exact, mode="hybrid") for _ in range(2))
    prompt(r, [90, 12, 150])
    decode(r, 1, 2, 3)
    r.evict(40, sinks=2, recent=10)
    others = [(s.weights.clone(), s.positions.clone()) for s in states(r)]
    r.seq_lens[2] = r.evicted[2] = 0                          # the engine gives the row away
    prompt(r, [0, 0, 70], seed=3), prompt(fresh, [0, 0, 70], seed=3)
    for s, f, (w, p) in zip(states(r), states(fresh), others):
        assert torch.equal(s.weights[2], f.weights[2]) and torch.equal(s.positions[2], f.positions[2])
        assert torch.equal(s.weights[:2], w[:2]) and torch.equal(s.positions[:2], p[:2])
    held, seen = list(r.seq_lens), [n + e for n, e in zip(r.seq_lens, r.evicted)]
    want = [evict64(s.weights.cpu(), s.positions.cpu(), held, seen, 30, 2, 10) for s in states(r)]
    r.evict(30, sinks=2, recent=10)
    for s, w in zip(states(r), want):
        assert torch.equal(s.weights.cpu(), w[4]) and torch.equal(s.positions.cpu(), w[5])
        for head in s.positions[2].cpu():
            assert {0, 1} | set(range(60, 70)) <= set(head[:30].tolist())


def test_a_sequence_of_one_token_starts_anew_in_a_decode_step(gpu):
    r = runner(gpu, exact_layers=2, mode="hybrid")
    prompt(r, [90, 12, 150])
    r.evict(40, sinks=2, recent=10)
    r.seq_lens[1] = r.evicted[1] = 0
    decode(r, 7, 8, 9)
    for s in states(r):
        assert (s.weights[1, :, 0] == G).all() and not s.weights[1, :, 1:].any()
        assert torch.equal(s.positions[1].cpu(), torch.arange(192, dtype=torch.int32).expand(2, 192))


def test_a_captured_step_starts_a_row_anew_too(gpu):
    r = runner(gpu, exact_layers=2, mode="full_tq")
    prompt(r, [20, 12, 30])
    for s in states(r):                                       # what an earlier sequence of the row would have left
        s.weights[1] = 5.0
        s.positions[1] = 99
    r.seq_lens[1] = 0
    replay, _ = r.capture_decode_step(190, torch.tensor([1, 2, 3], device=gpu))
    for step in range(3):
        replay(torch.tensor([4, step, 6], device=gpu))
        for s, got in zip(states(r), given(r)):
            assert torch.allclose(got, per_row(18 + step, 2 + step, 18 + step), rtol=1e-4)
            assert torch.equal(s.positions[1].cpu(), torch.arange(192, dtype=torch.int32).expand(2, 192))


def test_rows_in_another_order(gpu):
    a, b = (runner(gpu, exact_layers=1, mode="hybrid") for _ in range(2))
    for r in (a, b):
        prompt(r, [90, 12, 150])
        decode(r, 1, 2, 3)
        r.evict(40, sinks=2, recent=10)
        decode(r, 1, 2, 3)
    order = [2, 0, 1]
    batched.reorder_rows(b, order)
    b.block_table = b.block_table[order].contiguous()
    b.seq_lens, b.evicted = [b.seq_lens[i] for i in order], [b.evicted[i] for i in order]
    for s, t in zip(states(a), states(b)):
        assert torch.equal(s.weights[order], t.weights) and torch.equal(s.positions[order], t.positions)
    for r in (a, b):
        r.evict(30, sinks=2, recent=10)
    assert [a.seq_lens[i] for i in order] == b.seq_lens
    for s, t in zip(states(a), states(b)):
        assert torch.equal(s.weights[order], t.weights) and torch.equal(s.positions[order], t.positions)
    assert same(a.kv_caches, b.kv_caches) and same([s.pool.data for s in states(a)[1:]], [s.pool.data for s in states(b)[1:]])
    batched.reorder_rows(b, [1, -1, -1])
    for s, t in zip(states(a), states(b)):
        assert torch.equal(s.weights[0], t.weights[0]) and not t.weights[1:].any()       # (row 1 of [2, 0, 1] is a's row 0)
        assert torch.equal(t.positions[1].cpu(), torch.arange(192, dtype=torch.int32).expand(2, 192))
    kept = everything(b)
    for bad in ([0, 1], [0, 0, 1], [0, 1, 3], [0, 1, -2]):
        with pytest.raises(ValueError):
            batched.reorder_rows(b, bad)
    assert same(kept, everything(b))


def test_steps_of_fewer_rows_than_are_tracked_and_of_more(gpu):
    r, wide = runner(gpu, exact_layers=1, mode="hybrid"), runner(gpu, exact_layers=1, mode="hybrid", batch=5)
    for x in (r, wide):
        prompt(x, [90, 12, 150])
        decode(x, 1, 2, 3)
        x.evict(40, sinks=2, recent=10)
        decode(x, 1, 2, 3)
    assert r.seq_lens == wide.seq_lens
    for s, t in zip(states(r), states(wide)):
        assert torch.equal(s.weights, t.weights[:3]) and torch.equal(s.positions, t.positions[:3]) and not t.weights[3:].any()
    narrow = runner(gpu, exact_layers=1, mode="hybrid", batch=2)
    with pytest.raises(ValueError, match="rows"):
        prompt(narrow, [90, 12, 150])
    assert states(narrow)[0].tokens_written == 0 and not any(s.weights.any() for s in states(narrow))
    with pytest.raises(ValueError):
        evict_batched(narrow, narrow.block_table, torch.tensor([1, 1, 1], dtype=torch.int32, device=gpu), 40)


# ---- lengths ----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("exact", [0, 2])
def test_a_sequence_that_outgrows_what_is_tracked_is_refused(gpu, exact):
    r = runner(gpu, track=64, exact_layers=exact, mode="hybrid")
    with pytest.raises(ValueError, match="64"):
        prompt(r, [10, 12, 65])
    assert states(r)[0].tokens_written == 0 and not any(s.weights.any() for s in states(r))
    prompt(r, [10, 12, 63])
    decode(r, 1, 2, 3)
    kept = [t.clone() for s in states(r) for t in (s.weights, s.positions)]
    with pytest.raises(ValueError, match="64"):
        decode(r, 1, 2, 3)
    lens = torch.tensor([11, 13, 65], dtype=torch.int32)
    for bad in (dict(seq_lens=lens), dict(seq_lens=lens.to(gpu), max_len=65)):
        with pytest.raises(ValueError, match="64"):
            evict_batched(r, r.block_table, budget=20, **bad)
    assert all(torch.equal(a, b) for a, b in zip(kept, [t for s in states(r) for t in (s.weights, s.positions)]))
    r.evict(20)
    assert r.seq_lens == [11, 13, 20]
    decode(r, 1, 2, 3)


# ---- what is refused --------------------------------------------------------------------------------------------------------

def test_a_backend_that_writes_its_cache_in_forward_is_not_tracked(gpu):
    """Its blocks do not hold a step's tokens yet when the weights would be summed."""
    r = MinimalRunner(device=gpu, seed=5, **SIZE)
    for lay in r.layers:
        whole = lay.attn.impl

        class InForward:
            num_heads, num_kv_heads, head_size, scale, inner = whole.num_heads, whole.num_kv_heads, whole.head_size, whole.scale, whole

            def forward(self, layer, q, k, v, kv_cache, meta, *rest):
                self.inner.do_kv_cache_update(layer, k, v, kv_cache, meta.slot_mapping)
                return self.inner.forward(layer, q, k, v, kv_cache, meta, *rest)
        lay.attn.impl = InForward()
    install_batched_hooks(r, r.num_blocks, mode="capture_only")
    prompt(r, [20, 12, 30])
    with pytest.raises(ValueError, match="do_kv_cache_update"):
        track_weights(r, 3, 192)
    assert all(s.weights is None for s in states(r))
    decode(r, 1, 2, 3)


@pytest.mark.parametrize("exact", [0, 1, 2])
def test_a_cut_that_is_refused_leaves_everything_as_it_was(gpu, exact):
    r = runner(gpu, exact_layers=exact, mode="hybrid")
    prompt(r, [90, 12, 150])
    decode(r, 1, 2, 3)
    lens, table = torch.tensor(r.seq_lens, dtype=torch.int32, device=gpu), r.block_table
    kept = everything(r)
    for bad in (table.long(), table.cpu(), table[0], table[:2], table[:, :0]):
        with pytest.raises((ValueError, RuntimeError)):
            evict_batched(r, bad, lens, 40)
        with pytest.raises((ValueError, RuntimeError)):
            states(r)[0].evict(bad, lens, 40, kv_cache=r.kv_caches[0])
    for bad in (dict(seq_lens=lens[:2]), dict(seen=lens[:2]), dict(budget=0), dict(sinks=30, recent=30)):
        with pytest.raises(ValueError):
            evict_batched(r, table, **{**dict(seq_lens=lens, budget=40), **bad})
    last = r.layers[-1].attn                                  # (of all layers the one that would be cut last)
    whole = last.kv_cache
    for bad in ([torch.zeros(2, r.num_blocks, 8, 2, 64, dtype=torch.bfloat16, device=gpu)], [torch.zeros(2, 4, 16, 3, 64, dtype=torch.bfloat16, device=gpu)]):
        last.kv_cache = bad
        with pytest.raises(ValueError):
            evict_batched(r, table, lens, 40)
    assert same(kept, everything(r))
    last.kv_cache = whole
    r.evict(40)
    assert r.seq_lens == [40, 13, 40]


def test_an_exact_layer_without_its_cache_is_not_cut(gpu):
    r = runner(gpu, exact_layers=2, mode="hybrid")
    prompt(r, [90, 12, 150])
    lens, kept = torch.tensor(r.seq_lens, dtype=torch.int32, device=gpu), everything(r)
    with pytest.raises(ValueError, match="exact layer"):
        states(r)[0].evict(r.block_table, lens, 40)
    for bad in (None, [], [None], [r.kv_caches[-1][0]]):
        r.layers[-1].attn.kv_cache = bad
        with pytest.raises(ValueError, match="exact layer"):
            evict_batched(r, r.block_table, lens, 40)
    assert same(kept, everything(r))
    r.layers[-1].attn.kv_cache = r.kv_caches[-1]              # the tensor itself, not in a list
    assert evict_batched(r, r.block_table, lens, 40).tolist() == [40, 12, 40]


def test_a_decode_step_takes_memory_by_its_length_and_not_by_what_is_tracked(gpu):
    """Scores of every head and token of the step, not of every place for one: 3 x 8 heads of 400000 places would be 38 MB."""
    r = runner(gpu, track=400000, exact_layers=2, mode="hybrid")
    prompt(r, [90, 12, 150])
    s, q, meta = states(r)[0], torch.randn(3, 8, 64, device=gpu).bfloat16(), r.decode_metadata()
    meta.block_table = torch.nn.functional.pad(meta.block_table, (0, 25000))             # (an engine's rows have room for its longest sequence)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    s.attend(q, meta, kv_cache=r.kv_caches[0])
    assert torch.cuda.max_memory_allocated() - before < 1 << 20
    assert torch.allclose(given(r)[0], per_row(17, 13, 17), rtol=1e-4)
