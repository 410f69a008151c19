"""A hybrid step over a sequence that has been cut: what is exact in it are its last slots, which hold its newest tokens again only once as many have come."""

from types import SimpleNamespace

import pytest
import torch

from oracle import tq_oracle as O
from tests.helpers import cosine, key_code, params_of, value_code
from turboquant_amd.integration import vllm as single
from turboquant_amd.integration.batched import evict_batched, install_batched_hooks, track_weights
from turboquant_amd.integration.harness import MinimalRunner

pytestmark = pytest.mark.gpu

RING = 16


def expected(s, cache, table, q, lens):
    """Slots before the last RING from the pages, those from the engine's blocks, by the oracle."""
    out = []
    for b, n in enumerate(lens):
        hist, H = max(0, n - RING), s.config.num_kv_heads
        kc = vc = None
        if hist:
            idx, sgn, norms, rn, vd, vs, vz = [t.cpu() for t in s.pool.export_flat(table[b], hist)]
            kc, vc = key_code(idx, sgn, rn, norms, s.quantizer.bits - 1), value_code(vd, vs, vz, s.pool.value_bits)
        t = torch.arange(hist, n)
        k, v = (cache[i].cpu()[table[b].cpu()[t // 16].long(), t % 16] for i in range(2))
        out.append(O.hybrid_attention(q[b:b + 1].cpu(), kc, vc, max(hist, O.MIN_HISTORY) if hist else 0, params_of(s.quantizer), H, k, v))
    return torch.cat(out)


def test_the_last_slots_are_exact_and_every_token_counts_once(gpu):
    before = single.get_mode()
    try:
        r = MinimalRunner(device=gpu, seed=5, n_layers=1, hidden=256, num_heads=8, num_kv_heads=2, head_dim=64, ffn=512, vocab=500, batch=3, max_seq_len=200)
        install_batched_hooks(r, r.num_blocks, mode="hybrid", ring_capacity=RING)
        track_weights(r, 3, 200)
    finally:
        single.set_mode(before)
    (s,), cache, table = r._tq_layer_states.values(), r.kv_caches[0], r.block_table
    g = torch.Generator(gpu).manual_seed(0)
    cache.copy_(torch.randn(cache.shape, generator=g, device=gpu))
    lens = torch.tensor([90, 12, 150], dtype=torch.int32, device=gpu)
    s.ingest_paged_cache(cache, table, lens)
    s.weights.copy_(torch.rand(s.weights.shape, generator=g, device=gpu))
    seen = lens.clone()
    lens = evict_batched(r, table, lens, 64, sinks=2, recent=24)
    assert lens.tolist() == [64, 12, 64]
    for b, n, had in ((0, 64, 90), (2, 64, 150)):
        for head in s.positions[b, :, :n].cpu():
            assert set(range(had - 24, had)) <= set(head.tolist())                     # the newest are all there ..
            assert not set(range(had - RING, had)) <= set(head[n - RING:].tolist())    # .. but not in the last slots
    for step in range(RING + 1):
        q = torch.randn(3, 8, 64, generator=g, device=gpu).bfloat16()
        meta = SimpleNamespace(seq_lens=lens, block_table=table, max_seq_len=int(lens.max()))
        got, want = s.attend(q, meta, kv_cache=cache, hybrid=True).cpu(), expected(s, cache, table, q, lens.tolist())
        for b in range(3):
            for h in range(8):
                assert cosine(got[b, h], want[b, h]) >= 0.9999, (step, b, h)
        k, v = (torch.randn(3, 2, 64, generator=g, device=gpu).bfloat16() for _ in range(2))
        lens = lens + 1
        slot = (lens - 1).long()
        at = table.long().gather(1, (slot // 16)[:, None])[:, 0], slot % 16
        cache[0][at], cache[1][at] = k, v
        s.write(k, v, SimpleNamespace(num_actual_tokens=3, max_query_len=1, max_seq_len=int(lens.max()), seq_lens=lens, block_table=table))
        seen += 1
    for b, (n, had) in enumerate(zip(lens.tolist(), seen.tolist())):
        for head in s.positions[b, :, :n].cpu():
            assert head[n - RING:].tolist() == list(range(had - RING, had))            # the newest are the last slots again
