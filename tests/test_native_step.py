"""The native host side of a step's operators against the Python methods it stands in front of: the same results bit for bit where it takes a
call, nothing done where it does not."""

import pytest
import torch

from tests.step_helpers import DTYPES, Step
from tests.test_native_host import _same, both      # noqa: F401  (a fixture)
from turboquant_amd.rotary import inverse_frequencies, rotate_heads

pytestmark = pytest.mark.gpu
FORMS = ["plain", "one table", "no bounds", "cpu lengths", "long starts", "negated", "gradient", "strided", "inference", "refused"]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp8"])
def test_attention(gpu, both, kind, form):      # noqa: F811
    s = Step([70, 300, 5], [4, 40, 1], 2, 64, "fp8" if kind == "fp8" else DTYPES[kind], DTYPES["bf16" if kind == "fp8" else kind])
    q, one, starts, table, lens = s.query(6).to(gpu), s.query(6)[:3].to(gpu), s.starts, s.table, s.seq_lens
    kw = dict(max_len=300, window=50, sinks=4)
    if form == "one table":
        table = table[1]
    elif form == "no bounds":
        kw = dict(scale=-0.3)
    elif form == "cpu lengths":
        lens = lens.cpu().long()
    elif form == "long starts":
        starts = starts.long()
    elif form == "negated":
        q, one = torch._neg_view(q), torch._neg_view(one)
    elif form == "gradient":
        q, one = q.requires_grad_(), one.requires_grad_()
    elif form == "strided":
        q, one = torch.cat([q, q], -1)[..., :64], torch.cat([one, one], -1)[..., :64]
    elif form == "refused":
        kw = dict(window=0)

    def run():
        with torch.inference_mode(form == "inference"):
            cache = s.cache()
            try:
                return cache.attention(q, starts, table, lens, max_rows=40, **kw), cache.decode_attention(one, table, lens, **kw)
            except (RuntimeError, ValueError) as e:
                return type(e).__name__
    a, b, taken, left = both(run)
    assert _same(a, b)
    assert (a == "RuntimeError") == (form == "gradient") and (a == "ValueError") == (form == "refused")
    if form in ("plain", "one table", "no bounds", "inference"):
        assert left == 0 and taken == 3


@pytest.mark.parametrize("form", ["plain", "one table", "cpu lengths", "long starts", "negated", "gradient", "strided", "odd", "inference", "its own memory"])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_write_and_read(gpu, both, dtype, form):      # noqa: F811
    lens, runs = ([70], [40]) if form == "one table" else ([70, 300, 5], [4, 40, 1])
    k, v = (torch.randn(45 if len(runs) > 1 else 40, 2, 64, generator=torch.Generator().manual_seed(i)).to(DTYPES[dtype]).to(gpu) for i in (1, 2))
    if form == "negated":
        k, v = torch._neg_view(k), torch._neg_view(v)
    elif form == "gradient":
        k = k.requires_grad_()
    elif form == "strided":
        k, v = torch.cat([k, k], -1)[..., :64], torch.cat([v, v], 1)[:, :2]
    elif form == "odd":
        k = torch.cat([k.flatten()[:1], k.flatten()])[1:].view(k.shape)

    def run():
        with torch.inference_mode(form == "inference"):
            s = Step(lens, runs, 2, 64, "fp8", torch.bfloat16)
            table, at, starts = s.table, s.seq_lens, s.starts
            if form == "one table":
                table = table[0]
            elif form == "cpu lengths":
                at = at.cpu().long()
            elif form == "long starts":
                starts = starts.long()
            cache = s.cache()
            key = cache.key_cache.view(torch.uint8).view(-1)[: k.numel() * k.element_size()].view(k.dtype).view(k.shape) if form == "its own memory" else k
            try:
                cache.write(key, v, starts, table, at)
            except (RuntimeError, ValueError) as e:
                return type(e).__name__
            return *cache.read(starts, table, at, rows=k.shape[0] + 5, dtype=DTYPES[dtype]), cache.key_scales.clone(), cache.key_cache.view(torch.uint8).clone()
    a, b, taken, left = both(run)
    assert _same(a, b)
    assert (a == "RuntimeError") == (form == "gradient") and (a == "ValueError") == (form == "its own memory")
    if form in ("plain", "one table", "strided", "inference"):
        assert left == 0 and taken == 3


@pytest.mark.parametrize("form", ["plain", "no weights", "int positions", "projection", "odd", "gradient", "negated", "heads apart", "inference", "refused"])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_rotation(gpu, both, dtype, form):      # noqa: F811
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(11, 8 * 64, generator=g).to(DTYPES[dtype]).to(gpu)
    q, k = qkv[:, :256].reshape(11, 4, 64), qkv[:, 256:384].reshape(11, 2, 64)
    pos, f, w = torch.arange(11, device=gpu) * 1000, inverse_frequencies(64, device=gpu), torch.rand(64, generator=g).to(DTYPES[dtype]).to(gpu)
    kw = dict(q_weight=w, k_weight=w)
    if form == "no weights":
        kw = dict(interleaved=True)
    elif form == "int positions":
        pos = pos.to(torch.int32)
    elif form == "projection":
        q, k = qkv[:, :256].view(11, 4, 64), qkv[:, 256:384].view(11, 2, 64)
    elif form == "odd":
        q = torch.cat([q.flatten()[:1], q.flatten()])[1:].view(q.shape)
    elif form == "gradient":
        k = k.clone().requires_grad_()
    elif form == "negated":
        q = torch._neg_view(q)
    elif form == "heads apart":
        q = q.transpose(0, 1).contiguous().transpose(0, 1)
    elif form == "refused":
        pos = pos.float()

    def run():
        with torch.inference_mode(form == "inference"):
            try:
                return rotate_heads(q, k, pos, f, eps=1e-5, **kw)
            except (RuntimeError, ValueError) as e:
                return type(e).__name__
    a, b, taken, left = both(run)
    assert _same(a, b)
    assert (a == "RuntimeError") == (form == "gradient") and (a == "ValueError") == (form == "refused")
    if form in ("plain", "no weights", "int positions", "projection", "heads apart", "inference"):
        assert left == 0 and taken == 1
