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
