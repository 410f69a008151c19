"""Calls of a step's operators that the documentation allows and that are easy to get wrong: no sequences, outputs in place, factors and blocks of no
size, workspaces with old contents."""

import math

import pytest
import torch

from tests.step_helpers import DTYPES, Step
from turboquant_amd import _ffi
from turboquant_amd.rotary import inverse_frequencies, rotate_heads

pytestmark = pytest.mark.gpu
KINDS = {"bf16": (torch.bfloat16, torch.bfloat16), "fp16": (torch.float16, torch.float16), "fp8": ("fp8", torch.bfloat16), "fp8 fp16": ("fp8", torch.float16)}


@pytest.fixture(params=["native", "python"])
def side(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(_ffi, "native", lambda: None)
    return request.param


@pytest.mark.parametrize("kind", list(KINDS))
def test_a_step_of_no_sequence(gpu, side, kind):
    """Rows of nobody: zeros, or left as they are in a given output; nothing is written."""
    s = Step([20], [3], 2, 64, *KINDS[kind])
    cache, q = s.cache(), s.query(4).to(gpu)
    starts, table, lens = s.starts[:1], s.table[:0], s.seq_lens[:0]
    for n_split in (None, 3):
        kw = {} if n_split is None else dict(n_split=n_split, max_len=4000)
        assert (cache.attention(q, starts, table, lens, **kw) == 0).all()
        out = torch.full_like(q, 5)
        assert (cache.attention(q, starts, table, lens, out=out, **kw) == 5).all()
    if kind.startswith("fp8"):
        k, v = cache.read(starts, table, lens, rows=3)
        assert k.shape == (3, 2, 64) and (k == 0).all() and (v == 0).all()
        held = [t.clone().view(torch.uint8) for t in cache.operands()]
        cache.write(k, v, starts, table, lens)
        assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(held, cache.operands()))


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_rotation_in_place_with_as_many_heads(gpu, side, dtype):
    """Each output over its own input, several rounds of heads a workgroup; the other way about is refused (tests/test_step_calls_host.py)."""
    rows, H, d = 1030, 40, 128
    g = torch.Generator().manual_seed(1)
    q, k = (torch.randn(rows, H, d, generator=g).to(DTYPES[dtype]).to(gpu) for _ in range(2))
    pos, f = torch.arange(rows, device=gpu), inverse_frequencies(d, device=gpu)
    want = rotate_heads(q, k, pos, f)
    for out in ((q.clone(), k.clone()), (torch.empty_like(q), k.clone())):
        src = (out[0] if torch.equal(out[0], q) else q, out[1])
        got = rotate_heads(*src, pos, f, out=out)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(ValueError):
        rotate_heads(q, k, pos, f, out=(k, q))


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_one_row_of_any_stride(gpu, side, dtype):
    from turboquant_amd.fp8 import Fp8PagedCache
    x = torch.randn(4096, generator=torch.Generator().manual_seed(2)).to(DTYPES[dtype]).to(gpu)
    odd, even = x.as_strided((1, 2, 64), (1001, 64, 1)), x[:128].view(1, 2, 64).clone()
    pos, f = torch.tensor([12345], device=gpu), inverse_frequencies(64, device=gpu)
    assert all(torch.equal(a, b) for a, b in zip(rotate_heads(odd, odd, pos, f), rotate_heads(even, even, pos, f)))
    starts, table, lens = (torch.tensor(t, dtype=torch.int32, device=gpu) for t in ([0, 1], [[1]], [7]))
    held = []
    for t in (odd, even):
        cache = Fp8PagedCache.allocate(2, 2, 64, gpu)
        cache.write(t, t, starts, table, lens)
        held.append(cache)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(held[0].operands(), held[1].operands())) and held[0].key_scales.any()


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("G,runs", [(4, [1, 1]), (4, [3, 2]), (16, [2, 1]), (8, [40, 5])])
@pytest.mark.parametrize("scale", [1e-12, -1e-12, 1e-30, 1e-38])
def test_factors_of_no_size(gpu, kind, d, G, runs, scale):
    """Keys of zeros, whose 8-bit scales are the smallest there are, times a factor so small that the two are nothing together: all visible tokens
    have the same weight, and those behind the rows none."""
    s = Step([37, 70], runs, 2, d, *KINDS[kind])
    for b, n in enumerate(s.lens):
        blocks = s.table_cpu[b, : (n + 15) // 16].long()
        s.q[0].view(torch.uint8)[blocks.to(gpu)] = 0
        s.k64[blocks] = 0
        if kind.startswith("fp8"):
            s.scales[0][blocks.to(gpu)] = 10 if b else 0
    q = s.query(2 * G)
    s.check(q, s.cache().attention(q.to(gpu), s.starts, s.table, s.seq_lens, scale=scale), scale)
    s.check(q, s.cache().attention(q.to(gpu), s.starts, s.table, s.seq_lens, scale=scale, window=20, sinks=3), scale, 20, 3)


@pytest.mark.parametrize("lens,most", [([70, 300, 5], None), ([70, 300, 5], 64), ([70, 300, 0, 33], 1000), ([40], 1), ([], None), ([4200] + [20] * 30, None)])
def test_ingesting_into_8_bits(gpu, lens, most):
    """What the engine's blocks hold, the first tokens of every sequence: as one write of each sequence alone, and nothing else."""
    from turboquant_amd.fp8 import Fp8PagedCache
    from turboquant_amd.integration.batched import BatchedLayerState
    s = Step(lens or [5], [1] * max(1, len(lens)), 2, 64, torch.bfloat16, torch.bfloat16)
    kv = torch.stack([x.nan_to_num() for x in s.q])
    state = BatchedLayerState(config=None, quantizer=None, pool=None, fp8=Fp8PagedCache.allocate(s.blocks, 2, 64, gpu))
    state.ingest_paged_cache(kv, s.table, torch.tensor(lens, dtype=torch.int32), max_tokens=most)
    want = Fp8PagedCache.allocate(s.blocks, 2, 64, gpu)
    took = [n if most is None else min(n, most) for n in lens]
    for b, n in enumerate(took):
        t = torch.arange(n)
        at = s.table_cpu[b, t // 16].long().to(gpu), (t % 16).to(gpu)
        step = torch.tensor([0, n, n], dtype=torch.int32, device=gpu)
        want.write(kv[0][at], kv[1][at], step[:2], s.table[b: b + 1], step[2:])
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(state.fp8.operands(), want.operands()))
    assert state.tokens_written == sum(took)


def test_ingesting_more_than_the_table_holds(gpu):
    """Tokens without a block are left out."""
    from turboquant_amd.fp8 import Fp8PagedCache
    from turboquant_amd.integration.batched import BatchedLayerState
    s = Step([40, 30], [1, 1], 2, 64, torch.bfloat16, torch.bfloat16)
    kv = torch.stack([x.nan_to_num() for x in s.q])
    table = torch.tensor([[2, -1, 1], [3, s.blocks, 0]], dtype=torch.int32, device=gpu)
    held = []
    for lens in ([48, 48], [1000, 50]):
        state = BatchedLayerState(config=None, quantizer=None, pool=None, fp8=Fp8PagedCache.allocate(s.blocks, 2, 64, gpu))
        state.ingest_paged_cache(kv, table, torch.tensor(lens))
        held.append(state.fp8)
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(held[0].operands(), held[1].operands()))
    assert [int(x) > 0 for x in held[0].key_scales[:, 0]][:4] == [True] * 4 and not held[0].key_scales[4:].any()
