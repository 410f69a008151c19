"""Exact layers, weights and eviction together, the way an engine uses them: prompts, decode steps, a cut, decode steps, another cut."""

import pytest
import torch

from tests.exact_helpers import evict64
from turboquant_amd.integration import vllm as single
from turboquant_amd.integration.batched import evict_batched, get_batched_stats, install_batched_hooks, track_weights
from turboquant_amd.integration.harness import MinimalRunner

pytestmark = pytest.mark.gpu

SIZE = dict(n_layers=3, hidden=256, num_heads=8, num_kv_heads=2, head_dim=64, ffn=512, vocab=500, batch=3, max_seq_len=200)


def runner(gpu, **hooks):
    r = MinimalRunner(device=gpu, seed=5, **SIZE)
    if hooks:
        install_batched_hooks(r, r.num_blocks, **hooks)
    return r


@pytest.fixture(autouse=True)
def mode_back():
    before = single.get_mode()
    yield
    single.set_mode(before)


def prompt(r, lens, seed=0):
    toks = torch.randint(0, SIZE["vocab"], (sum(lens),), generator=torch.Generator().manual_seed(seed)).to(r.device)
    return r.step(toks, r.metadata(lens))


def near(a, b):
    """Logits of two exact paths in bf16: the same sums in another order, rounded at every layer."""
    return float((a.double() - b.double()).norm() / b.double().norm()) < 0.02


@pytest.mark.parametrize("mode", ["hybrid", "full_tq"])
def test_exact_layers_answer_as_the_engine_does(gpu, mode):
    plain, hooked = runner(gpu), runner(gpu, exact_layers=3, mode=mode)
    states = list(hooked._tq_layer_states.values())
    assert all(s.pool is None and s.memory_bytes() == 0 and not s.supports_hybrid for s in states)
    lens = [50, 3, 129]
    assert torch.equal(prompt(plain, lens), prompt(hooked, lens))
    for i in range(4):
        t = torch.tensor([i, 7 * i, 11], device=gpu)
        assert near(hooked.decode_step(t), plain.decode_step(t))
    assert get_batched_stats(hooked)["decode_steps"] == 4 and states[0].tokens_written == sum(lens) + 12
    assert single.free_kv_cache(hooked) == 0


def test_a_mix_of_exact_and_compressed_layers(gpu):
    plain, hooked = runner(gpu), runner(gpu, exact_layers=1, mode="hybrid", ring_capacity=1024)
    states = list(hooked._tq_layer_states.values())
    assert [s.pool is None for s in states] == [True, False, False]
    lens = [60, 20, 100]
    prompt(plain, lens), prompt(hooked, lens)
    t = torch.tensor([1, 2, 3], device=gpu)
    assert near(hooked.decode_step(t), plain.decode_step(t))      # the ring holds every token: all exact
    assert single.free_kv_cache(hooked) > 0 and hooked.kv_caches[0].dim() == 5 and hooked.kv_caches[1].dim() != 5


def test_prompts_decode_cuts_and_decode(gpu):
    """The cut cache is the engine's: a plain backend over the same blocks and lengths gives the same logits."""
    plain, hooked = runner(gpu), runner(gpu, exact_layers=3, mode="hybrid")
    track_weights(hooked, 3, 192, window=16)
    states = list(hooked._tq_layer_states.values())
    lens, G = [90, 12, 150], 4
    assert torch.equal(prompt(plain, lens), prompt(hooked, lens))
    for s in states:
        given = s.weights.sum(-1).cpu()                       # each of the newest queries gives 1 per head
        assert torch.allclose(given, torch.tensor([16.0, 12.0, 16.0])[:, None].expand(3, 2) * G, rtol=1e-4)
    for step in range(12):
        t = torch.tensor([step, 3 * step, 40], device=gpu)
        a, b = hooked.decode_step(t), plain.decode_step(t)
        assert near(a, b), step
        if step in (3, 7, 8):
            held, seen = list(hooked.seq_lens), [n + e for n, e in zip(hooked.seq_lens, hooked.evicted)]
            want = [evict64(s.weights.cpu(), s.positions.cpu(), held, seen, 64, 2, 20) for s in states]
            hooked.evict(64, sinks=2, recent=20)
            assert hooked.seq_lens == [min(n, 64) for n in held] and [n + e for n, e in zip(hooked.seq_lens, hooked.evicted)] == seen
            for s, w in zip(states, want):
                assert torch.equal(s.weights.cpu(), w[4]) and torch.equal(s.positions.cpu(), w[5])
                for row, n, had in zip(s.positions.cpu(), hooked.seq_lens, seen):
                    for head in row:
                        kept = set(head[:n].tolist())
                        assert {0, 1} <= kept and set(range(had - min(20, n), had)) <= kept
            for mine, theirs in zip(hooked.kv_caches, plain.kv_caches):
                theirs.copy_(mine)
            plain.seq_lens, plain.evicted = list(hooked.seq_lens), list(hooked.evicted)
    for s in states:
        assert (s.weights.cpu()[:, :, :].sum(-1) > 0).all() and not s.weights[:, :, 80:].any()


def test_pages_and_blocks_are_cut_alike(gpu):
    """Compressed layers: after a cut every page holds what quantising the cut blocks gives."""
    r = runner(gpu, mode="hybrid", ring_capacity=16)
    track_weights(r, 3, 192)
    prompt(r, [90, 12, 150])
    t = torch.tensor([1, 2, 3], device=gpu)
    r.decode_step(t)
    r.evict(48, recent=16)
    assert r.seq_lens == [48, 13, 48]
    for (name, s), cache in zip(r._tq_layer_states.items(), r.kv_caches):
        held = [s.pool.export_flat(r.block_table[b], n) for b, n in enumerate(r.seq_lens)]
        s.pool.data.zero_()
        s.ingest_paged_cache(cache, r.block_table, torch.tensor(r.seq_lens))
        for b, n in enumerate(r.seq_lens):
            for x, y in zip(held[b], s.pool.export_flat(r.block_table[b], n)):
                assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), name
    assert torch.isfinite(r.decode_step(t)).all()


def test_a_chunked_prompt_adds_up(gpu):
    """A prompt in two steps: the newest queries of both have a say, the second step's about the first step's tokens too."""
    r = runner(gpu, exact_layers=3, mode="capture_only")
    track_weights(r, 3, 192, window=8)
    prompt(r, [20, 10, 30])
    prompt(r, [5, 9, 40], seed=1)
    s = next(iter(r._tq_layer_states.values()))
    assert torch.allclose(s.weights.sum(-1).cpu(), torch.tensor([13.0, 16.0, 16.0])[:, None].expand(3, 2) * 4, rtol=1e-4)


def test_a_captured_step_adds_weights_and_ends_with_a_cut(gpu):
    eager, captured = (runner(gpu, exact_layers=3, mode="full_tq") for _ in range(2))
    for r in (eager, captured):
        track_weights(r, 3, 192, window=16)
        prompt(r, [50, 12, 90])
    t = torch.tensor([1, 2, 3], device=gpu)
    replay, first = captured.capture_decode_step(190, t)
    assert near(first, eager.decode_step(t))
    for step in range(3):
        t = torch.tensor([step, 9, 40 * step], device=gpu)
        assert near(replay(t), eager.decode_step(t)), step
        assert captured.seq_lens == eager.seq_lens
        for r in (eager, captured):
            for s in r._tq_layer_states.values():
                given = s.weights.sum(-1).cpu()               # every query so far gave 1 per head
                assert torch.allclose(given, torch.tensor([18.0 + step, 14.0 + step, 18.0 + step])[:, None].expand(3, 2) * 4, rtol=1e-4)
    captured.evict(48, sinks=4, recent=16)
    with pytest.raises(RuntimeError, match="cut"):
        replay(t)
    with pytest.raises(RuntimeError, match="cut"):
        captured.capture_decode_step(190, t)


def test_refusals(gpu):
    with pytest.raises(ValueError):
        runner(gpu, exact_layers=1, no_alloc=True, mode="full_tq")
    r = runner(gpu, mode="hybrid")
    with pytest.raises(RuntimeError):
        evict_batched(r, r.block_table, torch.tensor([0, 0, 0], dtype=torch.int32, device=gpu), 10)
    for window in (0, 1025):
        with pytest.raises(ValueError):
            track_weights(r, 3, 192, window=window)
    exact = runner(gpu, exact_layers=3, mode="hybrid")
    s = next(iter(exact._tq_layer_states.values()))
    with pytest.raises(RuntimeError):
        s.ingest_paged_cache(exact.kv_caches[0], exact.block_table, torch.tensor([1, 1, 1]))
    bare = MinimalRunner(device=gpu, seed=5, exact_cache=False, **SIZE)
    install_batched_hooks(bare, bare.num_blocks, mode="full_tq", no_alloc=True)
    with pytest.raises(ValueError):
        track_weights(bare, 3, 192)
