"""16-bit decode attention over the exact cache: the softmax weights of the value product are no coarser than the sums that they go into.

Scores are exact here up to two roundings: queries and keys hold -1, 0 and 1, so that q . k is a whole number in fp32 whatever the order of its additions.
What is left is the weights' own rounding, which 64 bits without it then show."""

import math

import pytest
import torch

from tests.exact_helpers import DTYPES, STEP32, Sequences, half_step

pytestmark = pytest.mark.gpu


def whole(*shape, seed):
    return torch.randint(-1, 2, shape, generator=torch.Generator().manual_seed(seed)).double()


def check(dtype, d, heads, H, lens, scale, **kw):
    from turboquant_amd.exact import ExactPagedCache
    dt = DTYPES[dtype]
    seqs = Sequences(lens, H, d, dt, seed=d + heads)
    for b, n in enumerate(lens):
        t = torch.arange(n)
        k = whole(n, H, d, seed=b)
        seqs.kv[0][seqs.table[b].cpu()[t // 16].long(), t % 16] = k.to(dt).to(seqs.device)
        seqs.k64[b] = k
    q = whole(len(lens), heads, d, seed=99)
    out = ExactPagedCache.from_engine(seqs.kv).decode_attention(q.to(dt).to(seqs.device), seqs.table, seqs.seq_lens, scale=scale, **kw).cpu().double()
    G, step = heads // H, half_step(dt)
    for b, n in enumerate(lens):
        k, v = (x[b].repeat_interleave(G, 1).transpose(0, 1) for x in (seqs.k64, seqs.v64))                       # (heads, n, d)
        s = (k @ q[b][:, :, None])[..., 0] * scale
        p = torch.softmax(s, -1)[:, None]
        want, size = (p @ v)[:, 0], (p @ v.abs())[:, 0]
        # A weight's logarithm: scale log2 e rounded twice, the product with it, the difference to the maximum, each half a step of what is at most twice the
        # largest score's; the same once more in the sum.  Its exponential, the sum of n weights and the products: n + 64 half steps.  The weight as
        # a high and a low half of the cache's type: the high one is cut, which leaves less than a whole step, and of that the low one is off by half a
        # step (2 step^2); below fp16's normal numbers by half of 2^-24, where the largest weight is 2^6 at least.
        rel = 2 * 4 * STEP32 * 2 * math.log2(math.e) * float(s.abs().max()) + (n + 64) * STEP32 + 2 * step * step
        err = rel * size
        if dt == torch.float16:
            err = err + 2.0 ** -31 * p.amax(-1) * v.abs().sum(1)
        allowed = err + 1.01 * step * (want.abs() + err) + 1e-30
        off = (out[b] - want).abs()
        assert (off <= allowed).all(), f"sequence {b}: off by {float((off / allowed).max()):.3g} of what is allowed"


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d,heads,H", [(64, 8, 2), (128, 32, 8), (192, 5, 1), (256, 16, 2), (320, 16, 1), (576, 16, 1), (768, 7, 1)])
def test_sixteen_heads(gpu, dtype, d, heads, H):
    check(dtype, d, heads, H, [1, 40, 300, 1500], 1.5 / math.sqrt(d * 4 / 9))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d,heads", [(64, 70), (128, 128), (256, 40), (448, 32), (512, 100), (576, 128)])
@pytest.mark.parametrize("splits", [None, 1])
def test_dozens_of_heads(gpu, dtype, d, heads, splits):
    """(with a bound on the lengths at which they share their reads)"""
    check(dtype, d, heads, 1, [1, 40, 700], 1.5 / math.sqrt(d * 4 / 9), max_len=1 << 21, n_split=splits)
