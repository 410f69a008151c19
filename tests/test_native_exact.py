"""The native host side of the exact cache's operators against the Python methods it stands in front of: the same results bit for bit where
it takes a call, nothing done where it does not."""

import pytest
import torch

from tests.exact_helpers import DTYPES, Sequences
from tests.test_native_host import _same, both      # noqa: F401  (a fixture)
from turboquant_amd.eviction import select_evictions
from turboquant_amd.exact import ExactPagedCache

pytestmark = pytest.mark.gpu

FORMS = ["plain", "one table", "no bound", "cpu lengths", "long table rows", "negated", "gradient", "strided weights", "rows apart", "inference",
         "expanded weights"]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("form", FORMS)
def test_decode_and_window(gpu, both, dtype, form):      # noqa: F811
    seqs = Sequences([70, 300, 5], 2, 64, DTYPES[dtype])
    q, rows = seqs.query(3, 8, 64).to(gpu), seqs.query(30, 8, 64, seed=3).to(gpu)
    starts = torch.tensor([0, 10, 29, 30], dtype=torch.int32, device=gpu)
    table, lens, kw, window_kw = seqs.table, seqs.seq_lens, dict(max_len=300), dict(max_len=300)
    w0 = torch.rand(3, 2, 320, device=gpu, generator=torch.Generator(gpu).manual_seed(0))
    if form == "one table":
        table = table[1]
    elif form == "no bound":
        kw, window_kw = dict(scale=0.3), dict(scale=-0.3)
    elif form == "cpu lengths":
        lens = lens.cpu().long()
    elif form == "long table rows":
        table = torch.cat([table, table], 1)[:, : table.shape[1]]
    elif form == "negated":
        q, rows = torch._neg_view(q), torch._neg_view(rows)
    elif form == "rows apart":
        q, rows = torch.cat([q, q], -1)[..., :64], torch.cat([rows, rows], -1)[..., :64]
    elif form == "strided weights":
        w0 = torch.rand(2, 3, 640, device=gpu, generator=torch.Generator(gpu).manual_seed(0)).transpose(0, 1)[..., 100:420]
    elif form == "gradient":
        q, rows = q.requires_grad_(), rows.requires_grad_()
    elif form == "expanded weights":
        w0 = w0[:1].expand(3, 2, 320)

    def run():
        w = w0 if form == "expanded weights" else w0.clone(memory_format=torch.preserve_format)
        if form == "strided weights":
            w = torch.empty_strided(w0.shape, w0.stride(), device=gpu).copy_(w0)
        version = w._version
        cache = ExactPagedCache.from_engine(seqs.kv)
        try:
            out = cache.decode_attention(q, table, lens, weights=w, **kw)
            assert w._version > version
            alone = cache.decode_attention(q, table, lens, **kw)
            cache.add_window_weights(rows, starts, table, lens, w, 7, **window_kw)
            return out, alone, w.clone()
        except (RuntimeError, ValueError) as e:
            return type(e).__name__
    if form == "inference":
        with torch.inference_mode():
            def run():                                  # noqa: F811
                w = w0.clone()
                cache = ExactPagedCache.from_engine(seqs.kv)
                out = cache.decode_attention(q, table, lens, weights=w)
                cache.add_window_weights(rows, starts, table, lens, w, 7)
                return out, w
            a, b, taken, left = both(run)
    else:
        a, b, taken, left = both(run)
    assert _same(a, b)
    assert (a == "RuntimeError") == (form == "gradient") and (a == "ValueError") == (form == "expanded weights")
    if form in ("plain", "one table", "no bound", "strided weights", "inference"):
        assert left == 0 and taken >= 3
    if form == "negated":
        cache = ExactPagedCache.from_engine(seqs.kv)
        assert _same(a[1], cache.decode_attention(q.clone(), table, lens, **kw))


@pytest.mark.parametrize("L,budget", [(100, 40), (20000, 1000)])
@pytest.mark.parametrize("form", ["plain", "seen", "cpu lengths", "strided", "negated", "in place", "refused"])
def test_evict(gpu, both, L, budget, form):              # noqa: F811
    g = torch.Generator().manual_seed(L)
    w = torch.rand(2, 3, L, generator=g).to(gpu)
    pos = torch.arange(L, dtype=torch.int32).expand(2, 3, L).contiguous().to(gpu)
    lens, seen, recent = torch.tensor([L, budget + 3], dtype=torch.int32, device=gpu), None, 8
    seqs = Sequences([L, budget + 3], 3, 64, torch.bfloat16)
    if form == "seen":
        seen = lens + 100
    elif form == "cpu lengths":
        lens = lens.cpu()
    elif form == "strided":
        w, pos = w.transpose(0, 1).contiguous().transpose(0, 1), pos.transpose(0, 1).contiguous().transpose(0, 1)
    elif form == "negated":
        w = torch._neg_view(w)
    elif form == "refused":
        recent = budget

    def run():
        kv = seqs.kv.clone()
        cache = ExactPagedCache(kv[0], kv[1])
        try:
            out = (w.clone(), pos.clone()) if form == "in place" else None
            e = select_evictions(*(out or (w, pos)), lens, budget, seen=seen, recent=recent, out=out)
        except ValueError as err:
            return str(err)
        version = kv._version
        cache.move_tokens(e, seqs.table)
        assert kv._version > version
        return tuple(e[:6]) + (e.budget, kv)
    a, b, taken, left = both(run)
    assert _same(a, b)
    if form in ("plain", "seen", "strided"):
        assert left == 0 and taken == 3


def test_a_cache_that_does_not_hold_its_values_is_refused(gpu):
    seqs = Sequences([40], 2, 64, torch.bfloat16)
    with pytest.raises(ValueError):
        ExactPagedCache(torch._neg_view(seqs.kv[0]), seqs.kv[1])
    w = torch._neg_view(torch.zeros(1, 2, 40, device=gpu))
    with pytest.raises(ValueError):
        ExactPagedCache.from_engine(seqs.kv).decode_attention(seqs.query(1, 4, 64).to(gpu), seqs.table, seqs.seq_lens, weights=w)
