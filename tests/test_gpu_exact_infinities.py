"""Decode attention over the exact cache where values are infinite: a weight times infinity is infinity, however the tokens are split and the weight is rounded."""

import math

import pytest
import torch

from tests.exact_helpers import DTYPES, Sequences

pytestmark = pytest.mark.gpu


def infinite(gpu, dtype, d, heads, seed, where, **kw):
    """One KV head of 600 tokens, weights between 1 and 2^-14 of the largest, powers of two among them; channel c of token where[c] is infinite."""
    from turboquant_amd.exact import ExactPagedCache
    dt, n = DTYPES[dtype], 600
    g = torch.Generator().manual_seed(seed)
    seqs = Sequences([n], 1, d, dt, seed=seed)
    t = torch.arange(n)
    k, v = torch.zeros(n, 1, d), torch.randn(n, 1, d, generator=g)
    k[:, 0, 0] = torch.randint(-7, 1, (n,), generator=g).float()
    k[0] = 0
    v[where, 0, torch.arange(d)] = math.inf
    for i, x in enumerate((k, v)):
        seqs.kv[i][seqs.table[0].cpu()[t // 16].long(), t % 16] = x.to(dt).to(gpu)
    q = torch.zeros(1, heads, d)
    q[0, :, 0] = torch.linspace(0.25, 2, heads)
    return ExactPagedCache.from_engine(seqs.kv).decode_attention(q.to(dt).to(gpu), seqs.table, seqs.seq_lens, scale=math.log(2), **kw)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("splits", [1, 2, 3, 7, 16, 19])
def test_in_any_part_of_a_sequence(gpu, dtype, splits):
    for at in (0, 300, 599):
        out = infinite(gpu, dtype, 64, 4, at, torch.full((64,), at), n_split=splits)
        assert (out == math.inf).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d,heads,bound", [(64, 4, 600), (128, 48, 1 << 21), (576, 100, 1 << 21)])
def test_whatever_its_weight(gpu, dtype, d, heads, bound):
    """A weight goes into the product as two 16-bit numbers: neither may be zero or negative, for weights that the type holds as for others."""
    for seed in range(4):
        where = torch.randint(0, 600, (d,), generator=torch.Generator().manual_seed(9 + seed))
        where[0] = 0
        assert (infinite(gpu, dtype, d, heads, seed, where, max_len=bound) == math.inf).all()
