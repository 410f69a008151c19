"""A paged exact cache with sequences in it, and decode attention over it in 64 bits with bounds on what 32 bits may be off."""

import math

import torch

PAGE = 16
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
STEP32 = 2.0 ** -24                        # half a step of fp32, relative


def half_step(dt):
    return torch.finfo(dt).eps / 2


class Sequences:
    """`lens` tokens each, in blocks handed out in no order; layout "engine" (blocks, 16, H, d), "heads" (blocks, H, 16, d) seen as
    such, or "padded": rows further apart than they are long.  Slots that hold no token are NaN."""

    def __init__(self, lens, H, d, dtype, seed=0, layout="engine", device="cuda", extra_blocks=3, width=None):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.H, self.d, self.dtype, self.device = list(lens), H, d, dtype, device
        pages = [(n + PAGE - 1) // PAGE for n in lens]
        self.blocks = sum(pages) + extra_blocks
        order = torch.randperm(self.blocks, generator=g).to(torch.int32)
        self.width = max(1, *pages) if width is None else width
        table = torch.full((len(pages), self.width), -1, dtype=torch.int32)
        self.k64, self.v64 = [], []
        flat = torch.full((2, self.blocks, PAGE, H, d), float("nan"), dtype=torch.float64)
        at = 0
        for b, (n, p) in enumerate(zip(lens, pages)):
            table[b, :p] = order[at: at + p]
            at += p
            kv = torch.randn(2, n, H, d, generator=g, dtype=torch.float64).to(dtype).double()
            self.k64.append(kv[0])
            self.v64.append(kv[1])
            t = torch.arange(n)
            flat[:, table[b, t // PAGE].long(), t % PAGE] = kv
        self.table = table.to(device)
        self.seq_lens = torch.tensor(self.lens, dtype=torch.int32, device=device)
        kv = flat.to(dtype).to(device)
        if layout == "heads":
            kv = kv.transpose(2, 3).contiguous().transpose(2, 3)
        elif layout == "padded":
            wide = torch.full((2, self.blocks, PAGE, H, d + 64), float("nan"), dtype=dtype, device=device)
            wide[..., :d] = kv
            kv = wide[..., :d]
        self.kv = kv

    def query(self, *shape, seed=1):
        return (2 * torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)).to(self.dtype)


def attention64(q, k, v, scale, keep=None):
    """One sequence: q (Hq, d), k / v (n, H, d) in 64 bits -> out (Hq, d), weights (H, n), and the bounds of both.

    A score is a sum of d products, off by at most (d + 4) half steps of fp32 times sum |q_i k_i| scale (the additions, the
    product with scale and log2 e); a weight's logarithm is off by twice that (its own score's and the sum's error).  exp2, the
    sum of n weights and their product's accumulation add at most n + 64 half steps, a weight rounded to the cache's
    16-bit type half a step of that; both act on sum p |v|."""
    Hq, d = q.shape
    n, H, _ = k.shape
    G = Hq // H
    q, kk, vv = q.double(), k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)          # (n, Hq, d)
    s = torch.einsum("hd,nhd->hn", q, kk) * scale
    if keep is not None:
        s = s.masked_fill(~keep, -math.inf)
        vv = vv.masked_fill(~keep[:, None, None], 0)
        kk = kk.masked_fill(~keep[:, None, None], 0)
    if n == 0 or (keep is not None and not keep.any()):
        return torch.zeros_like(q), torch.zeros(H, n, dtype=torch.float64), torch.zeros_like(q), torch.zeros(H, n, dtype=torch.float64)
    p = torch.softmax(s, -1)
    out = torch.einsum("hn,nhd->hd", p, vv)
    size = torch.einsum("hn,nhd->hd", p, vv.abs())
    score = (d + 4) * STEP32 * float((torch.einsum("hd,nhd->hn", q.abs(), kk.abs()) * abs(scale)).max())
    rel = 2 * score + (n + 64) * STEP32
    return out, p.view(H, G, n).sum(1), rel * size, rel * p.view(H, G, n).sum(1)


def check_decode(seqs, q, got, scale, weights_before=None, weights_after=None, keep=None, lens=None):
    """`got` (B, Hq, d) and the weights against 64 bits, element by element."""
    step = half_step(seqs.dtype)
    got = got.cpu()
    for b in range(got.shape[0]):
        n = seqs.lens[b] if lens is None else lens[b]
        kp = None if keep is None else keep[b][:n]
        out, w, out_err, w_err = attention64(q[b], seqs.k64[b][:n], seqs.v64[b][:n], scale, kp)
        if seqs.dtype != torch.float32:
            size = attention64(q[b], seqs.k64[b][:n], seqs.v64[b][:n].abs(), scale, kp)[0]
            out_err = out_err + 1.01 * step * size
        off = (got[b].double() - out).abs()
        allowed = out_err + step * (out.abs() + out_err) + 1e-30
        assert torch.isfinite(got[b]).all(), f"sequence {b}: not finite"
        assert (off <= allowed).all(), f"sequence {b} of {n}: off by {float((off / allowed).max()):.3g} of what is allowed"
        if weights_after is not None:
            L = weights_after.shape[2]
            before, after = weights_before[b].double(), weights_after[b].cpu().double()
            m = min(n, L)
            want = before.clone()
            want[:, :m] += w[:, :m]
            allowed = torch.zeros_like(want)
            allowed[:, :m] = w_err[:, :m] + 2 * STEP32 * (want[:, :m].abs() + w[:, :m])
            off = (after - want).abs()
            assert (off <= allowed).all(), f"weights of sequence {b}: off by {float((off / allowed.clamp_min(1e-30)).max()):.3g} of what is allowed"
