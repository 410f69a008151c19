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


def window64(seqs, q, starts, window, scale, keep=None, lens=None):
    """Weights (B, H, longest) that the newest `window` rows of q (rows, Hq, d) give in 64 bits, and their bound (attention64's for
    a weight; a sum over `rows` of them adds a half step each)."""
    lens = seqs.lens if lens is None else lens
    L = max(1, *lens)
    H, d = seqs.H, seqs.d
    out, err = (torch.zeros(len(lens), H, L, dtype=torch.float64) for _ in range(2))
    for b, n in enumerate(lens):
        run = max(0, min(starts[b + 1], q.shape[0]) - max(starts[b], 0))
        W = min(window, run, n)
        end = min(starts[b + 1], q.shape[0])
        for w in range(W):
            m = n - W + w + 1
            kp = None if keep is None else keep[b][:m]
            _, p, _, p_err = attention64(q[end - W + w], seqs.k64[b][:m], seqs.v64[b][:m], scale, kp)
            out[b, :, :m] += p
            err[b, :, :m] += p_err + W * q.shape[1] // H * STEP32 * p
    return out, err


def check_weights(got, before, add, err):
    L = got.shape[2]
    add, err = add[:, :, :L], err[:, :, :L]
    want = before.double().clone()
    want[:, :, : add.shape[2]] += add
    allowed = torch.zeros_like(want)
    allowed[:, :, : add.shape[2]] = err + 2 * STEP32 * (want[:, :, : add.shape[2]].abs() + add)
    off = (got.cpu().double() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= allowed).all(), f"off by {float((off / allowed.clamp_min(1e-30)).max()):.3g} of what is allowed"


def evict64(weights, positions, lens, seen, budget, sinks, recent):
    """select_evictions by its definition, sequence by sequence, on lists."""
    B, H, L = weights.shape
    new_w, new_p = torch.zeros_like(weights), torch.empty_like(positions)
    moves = max(1, min(budget, L - budget))
    count = torch.zeros(B, H, dtype=torch.int32)
    dst, src = (torch.full((B, H, moves), -1, dtype=torch.int32) for _ in range(2))
    left = []
    for b in range(B):
        n = max(0, min(int(lens[b]), L))
        had = int(lens[b]) if seen is None else int(seen[b])
        left.append(min(n, budget))
        for h in range(H):
            w, p = weights[b, h, :n].tolist(), positions[b, h, :n].tolist()

            def key(i):
                if p[i] < sinks or p[i] >= had - recent:
                    return 2, 0.0
                x = w[i]
                return 1, -math.inf if x != x else min(x, torch.finfo(torch.float32).max)
            kept = set(sorted(range(n), key=lambda i: (-key(i)[0], -key(i)[1], i))[:budget])
            holes = [i for i in range(min(n, budget)) if i not in kept]
            movers = [i for i in range(budget, n) if i in kept]
            assert len(holes) == len(movers)
            where = {i: i for i in kept if i < budget} | dict(zip(holes, movers))
            for to, of in where.items():
                new_w[b, h, to], new_p[b, h, to] = weights[b, h, of], positions[b, h, of]
            new_p[b, h, left[-1]:] = torch.arange(had, had + L - left[-1], dtype=torch.int32)
            count[b, h] = len(holes)
            dst[b, h, :len(holes)] = torch.tensor(holes, dtype=torch.int32)
            src[b, h, :len(holes)] = torch.tensor(movers, dtype=torch.int32)
    return torch.tensor(left, dtype=torch.int32), count, dst, src, new_w, new_p
