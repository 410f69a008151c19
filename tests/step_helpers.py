"""A step of rows over a paged cache - exact blocks, or e4m3 with a power of two per block and KV head -, and its results in 64 bits."""

import math

import torch

from tests.exact_helpers import DTYPES, PAGE, attention64, half_step      # noqa: F401
from turboquant_amd.exact import ExactPagedCache
from turboquant_amd.fp8 import Fp8PagedCache

LOWEST = -117
F8 = torch.float8_e4m3fn


def e4m3(x):
    """x (float64) to the nearest number of e4m3, ties to the even one, nothing beyond the largest; NaN stays."""
    step = torch.ldexp(torch.ones_like(x), (torch.frexp(torch.nan_to_num(x))[1] - 1).clamp_min(-6) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def exponents(x):
    """e (blocks, H) of blocks x (blocks, 16, H, d) in float64."""
    size = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax((1, 3))
    e = torch.full_like(size, LOWEST)
    for i in torch.arange(LOWEST, 120).tolist():
        e = torch.where(size > 448 * 2.0 ** i, torch.full_like(e, min(i + 1, 119)), e)
    return e


class Blocks8:
    """What an 8-bit cache holds, block by block, by the definition: q (blocks, 16, H, d) numbers of e4m3, e (blocks, H)."""

    def __init__(self, blocks, H, d):
        self.q, self.e = torch.zeros(blocks, PAGE, H, d, dtype=torch.float64), torch.full((blocks, H), -127.0, dtype=torch.float64)

    def write(self, x, block, first):
        """Rows x (n, H, d) to slots first .. of a block."""
        n = x.shape[0]
        new = torch.zeros(1, PAGE, *x.shape[1:], dtype=torch.float64)
        new[0, first: first + n] = x.double()
        e = exponents(new)[0]
        if first:
            was = self.e[block].clamp(LOWEST, 119)
            e = torch.maximum(e, was)
            self.q[block, :first] = e4m3(self.q[block, :first] * (2.0 ** (was - e))[:, None])
        self.e[block] = e
        self.q[block, first: first + n] = e4m3(x.double() / (2.0 ** e)[:, None])

    def values(self):
        return self.q * (2.0 ** self.e)[:, None, :, None]


class Step:
    """Sequences of `lens` tokens of which the last `runs` are the step's rows, in blocks handed out in no order; `extra` rows of no sequence behind
    them.  cache: a dtype of exact blocks, or "fp8".  Slots that hold no token are NaN."""

    def __init__(self, lens, runs, H, d, cache, dtype, seed=0, extra=0, spare=3, width=None, device="cuda", layout="engine"):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.runs, self.H, self.d, self.dtype, self.device, self.extra = list(lens), list(runs), H, d, dtype, device, extra
        pages = [(max(n, 0) + PAGE - 1) // PAGE for n in lens]
        self.blocks = sum(pages) + spare
        order = torch.randperm(self.blocks, generator=g).to(torch.int32)
        self.width = max(1, *pages) if width is None else width
        table = torch.full((len(pages), self.width), -1, dtype=torch.int32)
        at = 0
        for b, p in enumerate(pages):
            p = min(p, self.width)
            table[b, :p] = order[at: at + p]
            at += p
        k, v = (torch.randn(self.blocks, PAGE, H, d, generator=g, dtype=torch.float64) for _ in range(2))
        k = k * torch.exp(0.5 * torch.randn(H, d, generator=g, dtype=torch.float64))
        if cache == "fp8":
            held = []
            for x in (k, v):
                e = exponents(x)
                f = (2.0 ** e)[:, None, :, None]
                held.append((e4m3(x / f), e))
                x.copy_(held[-1][0] * f)
            q = [h[0].to(F8) for h in held]
            self.scales = [(h[1] + 127).to(torch.uint8).to(device) for h in held]
        else:
            q = [x.to(cache) for x in (k, v)]
            k, v = (x.double() for x in q)
        unused = torch.ones(self.blocks, PAGE, dtype=torch.bool)
        for b, n in enumerate(lens):
            t = torch.arange(min(max(n, 0), self.width * PAGE))
            unused[table[b, t // PAGE].long(), t % PAGE] = False
        for x in q:
            (x.view(torch.uint8) if cache == "fp8" else x)[unused] = 0x7f if cache == "fp8" else float("nan")
        q = [x.to(device) for x in q]
        if layout == "heads":
            q = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in q]
        elif layout == "padded":
            q = [torch.cat([x.view(torch.uint8), x.view(torch.uint8)[..., :64]], -1)[..., : x.view(torch.uint8).shape[-1]].view(x.dtype) for x in q]
        self.q = q
        self.table_cpu, self.k64, self.v64 = table, k, v
        self.table, self.seq_lens = table.to(device), torch.tensor(self.lens, dtype=torch.int32, device=device)
        self.starts = torch.tensor([0] + self.runs).cumsum(0).to(device=device, dtype=torch.int32)
        self.rows = sum(self.runs) + extra

    def cache(self):
        if self.q[0].dtype == F8:
            return Fp8PagedCache(*self.q, *self.scales)
        return ExactPagedCache(*self.q)

    def query(self, Hq, seed=1, size=1.0):
        g = torch.Generator().manual_seed(seed)
        return (size * torch.randn(self.rows, Hq, self.d, generator=g, dtype=torch.float64)).to(self.dtype)

    def tokens(self, b, n):
        """Keys and values (n, H, d) of sequence b's first n tokens, and whether they have a block in the cache."""
        t = torch.arange(n)
        page = t // PAGE
        block = torch.where(page < self.width, self.table_cpu[b, page.clamp_max(self.width - 1)], -torch.ones_like(page).to(torch.int32)).long()
        there = (block >= 0) & (block < self.blocks)
        at = block.clamp(0, self.blocks - 1)
        return self.k64[at, t % PAGE], self.v64[at, t % PAGE], there

    def check(self, q, got, scale, window=None, sinks=0, weight_step=None):
        """`got` (rows, Hq, d) against 64 bits, element by element: attention64's bound, a weight rounded to 16 bits (half a step of that type: weight_step)
        and the output's own rounding.  8 bits: the products' operands are the same numbers, and a score has one more product, with its block's
        scale, which is exact."""
        got, step = got.cpu(), half_step(self.dtype)
        weight_step = step if weight_step is None else weight_step
        assert got.dtype == self.dtype and torch.isfinite(got).all(), "not finite"
        row = 0
        for b, (n, run) in enumerate(zip(self.lens, self.runs)):
            k, v, there = self.tokens(b, max(n, 0))
            for i in range(run):
                p = n - run + i
                t = torch.arange(max(n, 0))
                seen = there & (t <= p)
                if window is not None:
                    seen &= (t > p - window) | (t < sinks)
                out, _, err, _ = attention64(q[row], k, v, scale, seen)
                size = attention64(q[row], k, v.abs(), scale, seen)[0]
                err = err + 1.01 * weight_step * size
                off, allowed = (got[row].double() - out).abs(), err + step * (out.abs() + err) + 1e-30
                assert (off <= allowed).all(), f"sequence {b} of {n}, row {i} of {run}: off by {float((off / allowed).max()):.3g} of what is allowed"
                row += 1


def rotate64(x, positions, inv_freq, weight, eps, interleaved):
    """rotate_heads by its definition, x (rows, H, d)."""
    x, r = x.double(), 2 * inv_freq.shape[0]
    if weight is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    angle = (positions.double()[:, None] * inv_freq)[:, None]
    cos, sin = angle.cos(), angle.sin()
    first = torch.arange(r // 2) * (2 if interleaved else 1)
    second = first + (1 if interleaved else r // 2)
    a, b = x[..., first], x[..., second]
    x = x.clone()
    x[..., first], x[..., second] = a * cos - b * sin, b * cos + a * sin
    return x
