"""Where the exact decode step may write its output."""

import pytest
import torch

from tests.exact_helpers import Sequences
from turboquant_amd.exact import ExactPagedCache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kw", [(4, dict(n_split=1)), (4, dict(n_split=3)), (40, dict(n_split=1)), (70, dict(max_len=1 << 21, n_split=1))])
def test_over_the_query_itself(gpu, heads, kw):
    seqs = Sequences([300, 5, 0], 1, 128, torch.bfloat16)
    cache, q = ExactPagedCache.from_engine(seqs.kv), seqs.query(3, heads, 128).to(gpu)
    want = cache.decode_attention(q, seqs.table, seqs.seq_lens, **kw)
    assert cache.decode_attention(q, seqs.table, seqs.seq_lens, out=q, **kw) is q
    assert torch.equal(q, want)


def test_over_a_part_of_what_is_read(gpu):
    """(a workgroup would write rows that another has yet to read)"""
    seqs = Sequences([300, 5, 40], 1, 128, torch.float32)
    cache = ExactPagedCache(seqs.kv[0], seqs.kv[1])
    q = torch.zeros(4, 4, 128, device=gpu)
    w = torch.zeros(3, 1, 4 * 128 * 3, device=gpu)
    call = lambda q, **kw: cache.decode_attention(q, seqs.table, seqs.seq_lens, **kw)
    for bad in (dict(q=q[:3], out=q[1:]), dict(q=q[:3], out=w.view(9, 4, 128)[2:5], weights=w), dict(q=q[:3], out=seqs.kv[0].reshape(-1)[:1536].view(3, 4, 128)),
                dict(q=q[:3], out=seqs.kv[1].reshape(-1)[:1536].view(3, 4, 128))):
        held = [t.clone() for t in (q, w, seqs.kv)]
        with pytest.raises(ValueError):
            call(**bad)
        assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(held, (q, w, seqs.kv)))
    call(q[:3], out=torch.empty(3, 4, 128, device=gpu), weights=w)
