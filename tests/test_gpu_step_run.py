"""A step's operators one behind the other, as a model's layer calls them, and as the batched hooks do: rotation, the cache's write, attention."""

import math

import pytest
import torch

from tests.exact_helpers import PAGE, attention64, half_step
from tests.step_helpers import Blocks8, rotate64
from turboquant_amd.fp8 import Fp8PagedCache
from turboquant_amd.integration import vllm as single
from turboquant_amd.integration.batched import install_batched_hooks, track_weights
from turboquant_amd.integration.harness import MinimalRunner
from turboquant_amd.rotary import inverse_frequencies, rotate_heads

pytestmark = pytest.mark.gpu

SIZE = dict(n_layers=3, hidden=256, num_heads=8, num_kv_heads=2, head_dim=64, ffn=512, vocab=500, batch=3, max_seq_len=200)


@pytest.fixture(autouse=True)
def mode_back():
    before = single.get_mode()
    yield
    single.set_mode(before)


def check_rows(q, got, held, lens, runs, scale, window=None, sinks=0):
    """got (rows, Hq, d) for the last runs[b] of lens[b] tokens of each sequence; held[b] its keys and values (lens[b], H, d) in 64 bits.  attention64's
    bound, a weight rounded to 16 bits and the output's own rounding."""
    row, step = 0, half_step(q.dtype)
    q, got = q.cpu(), got.cpu()
    assert torch.isfinite(got).all()
    for n, run, (k, v) in zip(lens, runs, held):
        for i in range(run):
            p, t = n - run + i, torch.arange(n)
            seen = t <= p
            if window is not None:
                seen &= (t > p - window) | (t < sinks)
            out, _, err, _ = attention64(q[row], k, v, scale, seen)
            err = err + 1.01 * step * attention64(q[row], k, v.abs(), scale, seen)[0]
            off, allowed = (got[row].double() - out).abs(), err + step * (out.abs() + err) + 1e-30
            assert (off <= allowed).all(), f"sequence of {n}, row {i} of {run}: off by {float((off / allowed).max()):.3g} of what is allowed"
            row += 1


def held_by(cache, table, lens):
    """Keys and values of each sequence as the 8-bit cache holds them."""
    starts = torch.tensor([0] + list(lens)).cumsum(0)
    k, v = cache.read(starts.to(cache.device), table, torch.tensor(lens, device=cache.device), rows=int(starts[-1]), dtype=torch.float32)
    cut = lambda x: x.cpu().double().split(list(lens))
    return list(zip(cut(k), cut(v)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window,sinks", [(None, 0), (24, 4)])
def test_a_layer(gpu, dtype, window, sinks):
    """A prompt in two chunks, sequences of different lengths, then single tokens: the projection's views rotated, written, attended to."""
    Hq, H, d, B = 8, 2, 128, 3
    g = torch.Generator().manual_seed(3)
    inv, weights = inverse_frequencies(d, theta=5e5), [(1 + 0.1 * torch.randn(d, generator=g)).to(dtype) for _ in range(2)]
    table = torch.randperm(B * 8, generator=g).to(torch.int32).view(B, 8)
    cache = Fp8PagedCache.allocate(B * 8, H, d, gpu)
    want = Blocks8(B * 8, H, d), Blocks8(B * 8, H, d)
    lens = [0] * B
    for runs in ([40, 7, 65], [30, 0, 3], [1, 1, 1], [1, 1, 1]):
        rows = sum(runs)
        lens = [n + r for n, r in zip(lens, runs)]
        starts = torch.tensor([0] + runs).cumsum(0).to(torch.int32)
        positions = torch.cat([torch.arange(n - r, n) for n, r in zip(lens, runs)])
        qkv = torch.randn(rows, (Hq + 2 * H) * d, generator=g).to(dtype)
        on = qkv.to(gpu)
        q, k, v = (x.view(rows, -1, d) for x in on.split([Hq * d, H * d, H * d], -1))
        rq, rk = rotate_heads(q, k, positions.to(gpu), inv.to(gpu), *(w.to(gpu) for w in weights))
        for x, y, w, heads in ((rq, q, weights[0], Hq), (rk, k, weights[1], H)):
            exact = rotate64(y.cpu(), positions, inv, w, 1e-6, False)
            # a head's norm and its turn: two products and their sum, off by some half steps of fp32 of the pair's size; one rounding to the output's type
            size = (exact[..., : d // 2].square() + exact[..., d // 2:].square()).sqrt().repeat(1, 1, 2)
            assert ((x.cpu().double() - exact).abs() <= half_step(dtype) * exact.abs() + (d + 32) * 2.0 ** -24 * size + 2.0 ** -24).all()
        table_on, lens_on, starts_on = table.to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu), starts.to(gpu)
        cache.write(rk, v, starts_on, table_on, lens_on)
        for x, held in ((rk.cpu(), want[0]), (v.cpu(), want[1])):
            for b, r in enumerate(runs):
                t = lens[b] - r
                while t < lens[b]:
                    end = min(lens[b], (t // PAGE + 1) * PAGE)
                    row = int(starts[b]) + t - (lens[b] - r)
                    held.write(x[row: row + end - t], int(table[b, t // PAGE]), t % PAGE)
                    t = end
        held = held_by(cache, table_on, lens)
        for b, n in enumerate(lens):
            t = torch.arange(n)
            for got, w in zip(held[b], want):
                assert torch.equal(got, w.values()[table[b, t // PAGE].long(), t % PAGE])
        if max(runs) == 1:
            got = cache.decode_attention(rq, table_on, lens_on, window=window, sinks=sinks)
        else:
            got = cache.attention(rq, starts_on, table_on, lens_on, window=window, sinks=sinks, max_rows=max(runs))
        check_rows(rq, got, held, lens, runs, 1 / math.sqrt(d), window, sinks)


class Recorder:
    """What each layer's attention is asked and answers."""

    def __init__(self, r):
        self.seen = []
        for lay in r.layers:
            lay.attn.impl.forward = self.around(lay.attn.impl.forward)

    def around(self, forward):
        def call(layer, q, k, v, cache, meta, *rest):
            got = forward(layer, q, k, v, cache, meta, *rest)
            self.seen.append((q.clone(), got.clone(), k.clone(), v.clone()))
            return got
        return call


def runner(gpu, exact_cache=True, window=None, sinks=0, qk_norm=True, hooks=True, **kw):
    r = MinimalRunner(device=gpu, seed=5, exact_cache=exact_cache, qk_norm=qk_norm, sliding_window=window, sink_tokens=sinks, **SIZE)
    if hooks:
        install_batched_hooks(r, r.num_blocks, **kw)
    return r


def step(r, runs, seed):
    toks = torch.randint(0, SIZE["vocab"], (sum(runs),), generator=torch.Generator().manual_seed(seed)).to(r.device)
    return r.decode_step(toks) if list(runs) == [1] * r.batch else r.step(toks, r.metadata(runs))


def rows_of(x, heads):
    return x.reshape(-1, heads, SIZE["head_dim"])


@pytest.mark.parametrize("mode", ["hybrid", "full_tq"])
@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 3)])
def test_hooked_layers(gpu, mode, window, sinks):
    """One layer exact, one in 8 bits, one in pages: prompts by the backend, single tokens from what each layer keeps."""
    r = runner(gpu, window=window, sinks=sinks, mode=mode, exact_layers=1, fp8_layers=1, initial_layers_count=0)
    exact, eight, pages = r._tq_layer_states.values()
    assert exact.fp8 is None and exact.pool is None and eight.pool is None and eight.fp8 is not None and pages.pool is not None
    assert exact.sees == eight.sees == (window, sinks) and pages.sees == (None, 0)
    assert eight.supports_hybrid and eight.memory_bytes() == eight.fp8.memory_bytes() == r.num_blocks * 2 * (16 * 2 * 64 + 2)
    rec = Recorder(r)
    lens = [0, 0, 0]
    for i, runs in enumerate(([50, 33, 5], [20, 1, 8], [1, 1, 1], [1, 1, 1])):
        rec.seen.clear()
        step(r, runs, i)
        lens = [n + x for n, x in zip(lens, runs)]
        held8 = held_by(eight.fp8, r.block_table, lens)
        if max(runs) > 1:
            continue
        t = [torch.arange(n) for n in lens]
        blocks = [(r.block_table[b].cpu().long()[t[b] // PAGE], t[b] % PAGE) for b in range(3)]
        held16 = [tuple(r.kv_caches[0][j].cpu()[at].double() for j in range(2)) for at in blocks]
        for (q, got, _, _), held in zip(rec.seen, (held16, held8)):
            check_rows(rows_of(q, 8), rows_of(got, 8), held, lens, runs, 1 / 8, window, sinks)
    assert eight.tokens_written == sum(lens) and eight.decode_steps == 2
    # what the engine's blocks of that layer hold, rounded block by block, is what its own hooks have written (its tokens in whole blocks)
    again = Fp8PagedCache.allocate(r.num_blocks, 2, 64, gpu)
    mine, eight.fp8 = eight.fp8, again
    eight.ingest_paged_cache(r.kv_caches[1], r.block_table, torch.tensor(lens))
    eight.fp8 = mine
    for b, n in enumerate(lens):
        at = (r.block_table[b].cpu().long()[torch.arange(n) // PAGE], torch.arange(n) % PAGE)
        for held, j in zip(held_by(again, r.block_table, lens)[b], range(2)):
            x = r.kv_caches[1][j].cpu()[at].double()
            size = torch.stack([x[i // PAGE * PAGE: i // PAGE * PAGE + PAGE].abs().amax((0, 2)) for i in range(n)])[..., None]
            # half a step of e4m3, and of what lies below its smallest normal number (2^-6 where the largest is 224 .. 448)
            assert ((held - x).abs() <= 2.0 ** -4 * x.abs() + 2.0 ** -10 / 224 * size).all()


@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 3)])
def test_prompts_without_the_engines_cache(gpu, window, sinks):
    """no_alloc: all layers in 8 bits, prompts in chunks, mixed steps and single tokens, captured ones too."""
    r = runner(gpu, exact_cache=False, window=window, sinks=sinks, mode="full_tq", no_alloc=True, fp8_layers=3)
    rec = Recorder(r)
    lens = [0, 0, 0]
    states = list(r._tq_layer_states.values())
    for i, runs in enumerate(([50, 33, 5], [20, 1, 8], [1, 1, 1])):
        rec.seen.clear()
        step(r, runs, i)
        lens = [n + x for n, x in zip(lens, runs)]
        for state, (q, got, _, _) in zip(states, rec.seen):
            check_rows(rows_of(q, 8), rows_of(got, 8), held_by(state.fp8, r.block_table, lens), lens, runs, 1 / 8, window, sinks)
    twin = runner(gpu, exact_cache=False, window=window, sinks=sinks, mode="full_tq", no_alloc=True, fp8_layers=3)
    for i, runs in enumerate(([50, 33, 5], [20, 1, 8], [1, 1, 1])):
        step(twin, runs, i)
    toks = [torch.tensor([7, 8 + i, 9], device=gpu) for i in range(4)]
    replay, first = r.capture_decode_step(180, toks[0])
    eager = twin.decode_step(toks[0])
    assert torch.equal(first, eager)
    for t in toks[1:]:
        torch.cuda.synchronize()
        got, want = replay(t), twin.decode_step(t)
        assert torch.equal(got, want)


def test_windowed_backend_and_hooks_agree(gpu):
    """The whole model: exact layers within a window against the backend's own answer, in the logits: bf16 rounds some eight times on a layer's way, half a step
    of 2^-8 each, three layers: 24 of them, a third of which would add up to 0.03 if all had one sign; without the window they differ by more than twice that."""
    a, b = (runner(gpu, window=16, sinks=2, hooks=h, **(dict(mode="hybrid", exact_layers=3) if h else {})) for h in (False, True))
    for i, runs in enumerate(([50, 33, 5], [1, 1, 1], [1, 1, 1])):
        x, y = step(a, runs, i).float(), step(b, runs, i).float()
        assert (x - y).norm() <= 0.03 * x.norm()
    full = runner(gpu, mode="hybrid", exact_layers=3)
    for i, runs in enumerate(([50, 33, 5], [1, 1, 1], [1, 1, 1])):
        z = step(full, runs, i).float()
    assert (x - z).norm() > 0.06 * x.norm()


def test_what_cannot_be_cut_is_refused(gpu):
    r = runner(gpu, mode="hybrid", fp8_layers=1)
    with pytest.raises(ValueError, match="8-bit layers cannot be cut"):
        track_weights(r, 3, 100)
    r = runner(gpu, window=20, mode="hybrid", exact_layers=1)
    with pytest.raises(ValueError, match="sliding window"):
        track_weights(r, 3, 100)
    assert all(s.weights is None for s in r._tq_layer_states.values())


@pytest.mark.parametrize("window,sinks", [(None, 0), (24, 4)])
def test_a_captured_layer_is_replayed(gpu, window, sinks):
    """Rotation, write and attention in one graph: every replay is another step (chunks, single tokens, rows of no sequence), the program's own work in between."""
    Hq, H, d, B, rows = 16, 2, 64, 3, 90
    g = torch.Generator().manual_seed(8)
    inv = inverse_frequencies(d, device=gpu)
    table = torch.randperm(B * 20, generator=g).to(torch.int32).view(B, 20).to(gpu)
    caches = [Fp8PagedCache.allocate(B * 20, H, d, gpu) for _ in range(2)]
    qkv = torch.zeros(rows, (Hq + 2 * H) * d, dtype=torch.bfloat16, device=gpu)
    positions, starts, lens = (torch.zeros(n, dtype=torch.int32, device=gpu) for n in (rows, B + 1, B))
    workspace = caches[0].workspace(rows, Hq, 320, B=B, max_rows=rows, window=window, sinks=sinks)

    def layer(cache, **kw):
        q, k, v = (x.view(rows, -1, d) for x in qkv.split([Hq * d, H * d, H * d], -1))
        q, k = rotate_heads(q, k, positions, inv)
        cache.write(k, v, starts, table, lens)
        return q, cache.attention(q, starts, table, lens, window=window, sinks=sinks, max_len=320, max_rows=rows, **kw)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(caches[0], workspace=workspace)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, out = layer(caches[0], workspace=workspace)
    now = [0] * B
    for runs in ([40, 17, 33], [1, 1, 1], [5, 0, 80], [60, 1, 2], [1, 1, 1]):
        now = [n + r for n, r in zip(now, runs)]
        qkv.copy_(torch.randn(qkv.shape, generator=g))
        starts.copy_(torch.tensor([0] + runs).cumsum(0))
        lens.copy_(torch.tensor(now))
        positions.copy_(torch.cat([torch.arange(n - r, n) for n, r in zip(now, runs)] + [torch.zeros(rows - sum(runs), dtype=torch.long)]))
        graph.replay()
        torch.cuda.synchronize()
        _, eager = layer(caches[1])
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and (out[sum(runs):] == 0).all()
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(caches[0].operands(), caches[1].operands()))
        check_rows(q[: sum(runs)], out[: sum(runs)], held_by(caches[0], table, now), now, runs, 1 / math.sqrt(d), window, sinks)
