"""What rounding the softmax's weights to 16 bits may cost: nothing where all tokens have the same values, and in decode steps, which go into the value product as two
halves, 2^-15 of a weight (fp16: 2^-21)."""

import math

import pytest
import torch

from tests.step_helpers import Step
from tests.test_gpu_attend import KINDS

pytestmark = pytest.mark.gpu


def same_values(s, seed=3):
    """All of a head's tokens get one vector of values, numbers of the cache's type; returned in 64 bits (H, d)."""
    g = torch.Generator().manual_seed(seed)
    if hasattr(s, "scales"):
        c = torch.randint(24, 104, (s.H, s.d), generator=g, dtype=torch.uint8)             # positive, of normal size
        s.scales[1].fill_(127)
        value = c.view(torch.float8_e4m3fn).double()
    else:
        c = (1 + torch.rand(s.H, s.d, generator=g)).to(s.q[1].dtype)
        value = c.double()
    for b, n in enumerate(s.lens):
        t = torch.arange(n)
        s.q[1].view(c.dtype)[s.table_cpu[b, t // 16].long().to(s.device), (t % 16).to(s.device)] = c.to(s.device)
    return value


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("G,runs", [(4, [2, 1, 5]), (4, [40, 33, 130]), (40, [5, 40, 7])])
def test_values_that_are_all_the_same(gpu, kind, d, G, runs):
    """Weights sum to one: numerators and sum are of the same weights, however they are rounded, so that the quotient is off by sums of n products in 32 bits (and by
    2^-15 where a weight is two halves), less than half a step of any output."""
    s = Step([5, 40, 1300], runs, 2, d, *KINDS[kind])
    c = same_values(s)
    q = s.query(2 * G, size=2.0).to(gpu)
    for kw in (dict(), dict(window=33, sinks=2), dict(n_split=3)):
        got = s.cache().attention(q, s.starts, s.table, s.seq_lens, **kw).cpu()
        want = c.to(got.dtype).repeat_interleave(G, 0).repeat(got.shape[0], 1, 1)
        want[: max(0, runs[0] - s.lens[0])] = 0               # (rows in front of the first token)
        assert torch.equal(got, want), f"off by {float(((got.double() - want.double()) / want.double()).abs().max()) * 2 ** 8:.3g} steps of bf16"
    got = s.cache().decode_attention(q[:3], s.table, s.seq_lens, window=1000).cpu()
    assert torch.equal(got, c.to(got.dtype).repeat_interleave(G, 0).expand_as(got))


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("G", [1, 16, 32, 33, 64, 128, 160])
def test_decode_steps_lose_nothing_by_their_heads(gpu, kind, d, G):
    """A decode step's weights are two halves whatever the number of heads on one."""
    s = Step([1, 70, 333, 0], [1] * 4, 1, d, *KINDS[kind])
    q = s.query(G)
    for window, sinks in ((20, 3), (1000, 0)):
        got = s.cache().decode_attention(q.to(gpu), s.table, s.seq_lens, window=window, sinks=sinks)
        s.check(q, got, 1 / math.sqrt(d), window, sinks, weight_step=2.0 ** -21 if kind == "fp16" else 2.0 ** -15)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("runs", [[2, 1, 3, 2], [12, 40, 20, 33]])
@pytest.mark.parametrize("n_split", [1, 3])
def test_a_sequence_alone_has_the_same_bits(gpu, kind, runs, n_split):
    """With a number of splits given, of the same tokens at most, and as many rows x heads that the same kernel answers (up to 16, up to 32, more), a sequence's rows do
    not depend on who else is in the step."""
    s = Step([500, 40, 77, 900], runs, 2, 64, *KINDS[kind])
    q, cache, longest = s.query(6).to(gpu), s.cache(), s.table.shape[1] * 16
    got = cache.attention(q, s.starts, s.table, s.seq_lens, n_split=n_split, max_rows=max(runs), max_len=longest)
    at = 0
    for b, run in enumerate(runs):
        alone = torch.tensor([0, run], dtype=torch.int32, device=gpu)
        one = cache.attention(q[at: at + run], alone, s.table[b: b + 1], s.seq_lens[b: b + 1], n_split=n_split, max_len=longest)
        assert torch.equal(one, got[at: at + run]), b
        at += run
