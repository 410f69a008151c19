"""Heads' norms and rotation against the definition in 64 bits."""

import pytest
import torch

from tests.step_helpers import DTYPES, half_step, rotate64
from turboquant_amd.rotary import inverse_frequencies, rotate_heads

pytestmark = pytest.mark.gpu
STEP32 = 2.0 ** -24


def inputs(rows, Hq, H, d, dtype, seed=0, furthest=1 << 20):
    g = torch.Generator().manual_seed(seed)
    q, k = (torch.randn(rows, n, d, generator=g).to(dtype) for n in (Hq, H))
    wq, wk = ((1 + 0.3 * torch.randn(d, generator=g)).to(dtype) for _ in range(2))
    return q, k, torch.randint(furthest, (rows,), generator=g), wq, wk


def check(got, x, positions, inv_freq, weight, eps, interleaved):
    """Sines, cosines and their arguments are off by 8 half steps of fp32 (the angle in turns is rounded to one of 1/2, times pi: 4, and the functions
    4); the norm's sum of d squares d + 8 of its own size, of which the square root halves the effect; two products and a sum; then the output's
    rounding.  All of it relative to the pair's size."""
    want = rotate64(x, positions, inv_freq, weight, eps, interleaved)
    y = rotate64(x, positions * 0, inv_freq, weight, eps, interleaved).abs()
    r, d = 2 * inv_freq.shape[0], x.shape[-1]
    size = y.clone()
    first = torch.arange(r // 2) * (2 if interleaved else 1)
    second = first + (1 if interleaved else r // 2)
    size[..., first] = size[..., second] = y[..., first] + y[..., second]
    err = (16 + (d + 8 if weight is not None else 0)) * STEP32 * size
    off = (got.cpu().double() - want).abs()
    allowed = err + half_step(x.dtype) * (want.abs() + err) + torch.finfo(x.dtype).tiny * torch.finfo(x.dtype).eps
    assert torch.isfinite(got).all() and (off <= allowed).all(), f"off by {float((off / allowed).max()):.3g} of what is allowed"


@pytest.mark.parametrize("d,r", [(64, 64), (128, 128), (128, 64), (192, 192), (192, 32), (256, 256), (256, 8), (8, 8), (72, 40), (512, 512), (128, 0)])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("norm,interleaved", [(True, False), (False, True), (True, True)])
def test_sizes(gpu, dtype, d, r, norm, interleaved):
    q, k, pos, wq, wk = inputs(13, 5, 2, d, DTYPES[dtype])
    f = inverse_frequencies(r)
    weights = (wq, wk) if norm else (None, None)
    got = rotate_heads(q.to(gpu), k.to(gpu), pos.to(gpu), f.to(gpu), *(None if w is None else w.to(gpu) for w in weights), interleaved=interleaved)
    check(got[0], q, pos, f, weights[0], 1e-6, interleaved)
    check(got[1], k, pos, f, weights[1], 1e-6, interleaved)


@pytest.mark.parametrize("rows", [1, 2, 1023, 1024, 1030])
@pytest.mark.parametrize("Hq,H", [(32, 8), (1, 1), (40, 0), (0, 3), (7, 2)])
def test_rows_and_heads(gpu, rows, Hq, H):
    q, k, pos, wq, wk = inputs(rows, Hq, H, 128, torch.bfloat16)
    f = inverse_frequencies(128, 500000.0)
    got = rotate_heads(q.to(gpu), k.to(gpu), pos.to(torch.int32).to(gpu), f.to(gpu), wq.to(gpu), None, eps=1e-5)
    check(got[0], q, pos, f, wq, 1e-5, False)
    check(got[1], k, pos, f, None, 1e-5, False)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_views_of_a_projection_and_in_place(gpu, dtype):
    q, k, pos, wq, wk = inputs(21, 4, 2, 64, DTYPES[dtype], seed=3)
    f = inverse_frequencies(64)
    qkv = torch.cat([q.flatten(1), k.flatten(1), k.flatten(1)], 1).to(gpu)
    vq, vk = qkv[:, :256].view(21, 4, 64), qkv[:, 256:384].view(21, 2, 64)
    args = pos.to(gpu), f.to(gpu), wq.to(gpu), wk.to(gpu)
    new = rotate_heads(vq, vk, *args)
    plain = rotate_heads(q.to(gpu), k.to(gpu), *args)
    assert all(torch.equal(a, b) for a, b in zip(new, plain)) and new[0].is_contiguous()
    version = qkv._version
    over = rotate_heads(vq, vk, *args, out=(vq, vk))
    assert over[0] is vq and qkv._version > version
    assert torch.equal(vq, plain[0]) and torch.equal(vk, plain[1]) and torch.equal(qkv[:, 384:], k.flatten(1).to(gpu))
    heads = q.to(gpu).transpose(0, 1).contiguous().transpose(0, 1), k.to(gpu)
    assert torch.equal(rotate_heads(*heads, *args)[0], plain[0])
    odd = torch.cat([q.flatten()[:1], q.flatten()])[1:].view(21, 4, 64).to(gpu)
    assert torch.equal(rotate_heads(odd, k.to(gpu), *args)[0], plain[0])
    assert torch.equal(rotate_heads(torch._neg_view(-q.to(gpu)), k.to(gpu), *args)[0], plain[0])


def test_far_and_negative_positions(gpu):
    q, k, _, _, _ = inputs(6, 2, 1, 128, torch.float32, seed=4)
    pos, f = torch.tensor([0, -5, (1 << 31) - 1, 1 << 33, -(1 << 30), 123456789]), inverse_frequencies(128)
    got = rotate_heads(q.to(gpu), k.to(gpu), pos.to(gpu), f.to(gpu))
    # an angle of up to 2^33 has a half step of 2^33 2^-53 in 64 bits: two of them here, one in the definition; the rest as in check
    want = rotate64(q, pos, f, None, 0.0, False)
    size = 2 * q.abs().max().double()
    assert ((got[0].cpu().double() - want).abs() <= (3 * 2.0 ** -20 + 20 * STEP32) * size).all()


def test_values_at_the_ends(gpu):
    """Zeros stay zeros with a norm; infinities and NaN stay in their head."""
    q, k, pos, wq, wk = inputs(3, 3, 1, 64, torch.bfloat16, seed=5)
    q[0, 0] = 0
    q[1, 1, 5], q[2, 2, 60] = float("inf"), float("nan")
    f = inverse_frequencies(32)
    got = rotate_heads(q.to(gpu), k.to(gpu), pos.to(gpu), f.to(gpu), wq.to(gpu), wk.to(gpu))[0].cpu()
    assert (got[0, 0] == 0).all()
    bad = torch.zeros(3, 3, dtype=torch.bool)
    bad[1, 1] = bad[2, 2] = True
    assert torch.isfinite(got[~bad]).all() and not torch.isfinite(got[1, 1]).all() and torch.isnan(got[2, 2]).any()
    plain = rotate_heads(q.to(gpu), k.to(gpu), pos.to(gpu), f.to(gpu))[0].cpu()
    assert torch.equal(plain[..., 32:].nan_to_num(7), q[..., 32:].nan_to_num(7))       # channels that do not turn are as they were


def test_captured(gpu):
    q, k, pos, wq, wk = (t.to(gpu) for t in inputs(9, 4, 2, 128, torch.bfloat16, seed=6))
    f = inverse_frequencies(128, device=gpu)
    rotate_heads(q, k, pos, f, wq, wk)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = rotate_heads(q, k, pos, f, wq, wk)
    for i in range(3):
        q.mul_(1.5); pos.add_(17)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, rotate_heads(q, k, pos, f, wq, wk)))
