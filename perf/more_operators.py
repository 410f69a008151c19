"""A cache in 8 bits, attention over it, windows, and what makes its keys, as timed cases.

A serving engine holds keys and values in blocks of 16 tokens that sequences reach through block tables.  A step has rows
query_start_loc[b] .. query_start_loc[b + 1] of sequence b, the last of them its token seq_lens[b] - 1.  A case is a dict of plain values; `kind` says
which operator it takes:

  store   a step's keys and values are written into the 8-bit cache (e4m3, a power of two for every block and KV head), and the blocks they went
          to are read back (`Fp8PagedCache.write`, `.read`)
  fp8     attention of a step's rows over that cache (`Fp8PagedCache.decode_attention`, `.attention`)
  exact   the same over the engine's exact blocks, within a sliding window and a few first tokens (`ExactPagedCache.decode_attention`, `.attention`)
  rotate  the norm of every head of queries and keys, and the rotation by position (`rotary.rotate_heads`)

With `own` false the same is computed by elementary torch operations in 32 bits.
"""

import math

import torch

own = False

PAGE = 16
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEVICE = "cuda:0"
F8 = torch.float8_e4m3fn
F8_MAX = 448.0
LOWEST = -117                  # exponent of the smallest scale: of a block of zeros


def listed():
    return [
        # ---- keys and values into 8 bits and back --------------------------------------------------------------------------
        # a decode step of a batch of chats: one token each, into blocks that are partly full
        dict(name="store_step", kind="store", seqs=64, shortest=500, longest=8000, rows=1, kv_heads=8, head_dim=128, dtype="bf16"),
        # four documents, all of a layer's tokens at once
        dict(name="store_prompts", kind="store", seqs=4, shortest=8192, longest=8192, rows=8192, kv_heads=8, head_dim=128, dtype="bf16"),
        # a mixed step: prompts of odd lengths and chunks that go on in the middle of a block, wide heads
        dict(name="store_ragged", kind="store", seqs=9, shortest=17, longest=4099, rows=777, kv_heads=2, head_dim=256, dtype="fp16"),
        # ---- attention over 8 bits -------------------------------------------------------------------------------------------
        # a chat's reply, one sequence in one layer: launches and latency are what counts
        dict(name="fp8_chat", kind="fp8", seqs=1, shortest=700, longest=700, rows=1, q_heads=32, kv_heads=8, head_dim=128, window=0, sinks=0,
             dtype="bf16"),
        # a batch of chats of a grouped-query model
        dict(name="fp8_batch", kind="fp8", seqs=32, shortest=8192, longest=8192, rows=1, q_heads=32, kv_heads=8, head_dim=128, window=0,
             sinks=0, dtype="bf16"),
        # one long document, wide heads, few of them
        dict(name="fp8_long", kind="fp8", seqs=1, shortest=131072, longest=131072, rows=1, q_heads=16, kv_heads=2, head_dim=256, window=0,
             sinks=0, dtype="bf16"),
        # a few drafted tokens of every sequence looked at together, sequences of very different length
        dict(name="fp8_drafts", kind="fp8", seqs=24, shortest=61, longest=16000, rows=5, q_heads=32, kv_heads=8, head_dim=128, window=0,
             sinks=0, dtype="fp16"),
        # chunks of two prompts behind what is written of them already
        dict(name="fp8_prompts", kind="fp8", seqs=2, shortest=8192, longest=8192, rows=2048, q_heads=32, kv_heads=8, head_dim=128, window=0,
             sinks=0, dtype="bf16"),
        # ---- windows ---------------------------------------------------------------------------------------------------------
        # a decode step of long sequences that look at the last 4096 tokens and the first four
        dict(name="window_step", kind="exact", seqs=32, shortest=30011, longest=32768, rows=1, q_heads=32, kv_heads=8, head_dim=128,
             window=4096, sinks=4, dtype="bf16"),
        # a whole prompt through such a layer
        dict(name="window_prompt", kind="exact", seqs=1, shortest=8192, longest=8192, rows=8192, q_heads=32, kv_heads=8, head_dim=128,
             window=4096, sinks=4, dtype="bf16"),
        # ---- norms and rotation ----------------------------------------------------------------------------------------------
        # a decode step of a batch, positions far out
        dict(name="rotate_step", kind="rotate", rows=64, q_heads=32, kv_heads=8, head_dim=128, rotary_dim=128, norm=True, interleaved=False,
             furthest=131072, dtype="bf16"),
        # the prompts of a step
        dict(name="rotate_prompts", kind="rotate", rows=16384, q_heads=40, kv_heads=8, head_dim=128, rotary_dim=128, norm=True,
             interleaved=False, furthest=16384, dtype="bf16"),
    ]


# ---- drawn cases ----------------------------------------------------------------------------------------------------------

def _between(rng, lo, hi):
    """A whole number spread over the logarithm of lo .. hi."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the same ranges, no more work than the largest listed ones, whose cache and plain form's scores fit the card."""
    most = [work(c) for c in listed()]
    while True:
        case = _draw(rng)
        w = work(case)
        if any(w[k] > max(m[k] for m in most) for k in ("bytes", "flops")) or w["bytes"] < 1e4:
            continue
        if case["kind"] != "rotate" and sum(_lengths(case)) * case["kv_heads"] * case["head_dim"] > 2 ** 30:
            continue
        if case["kind"] in ("fp8", "exact") and case["seqs"] * case["q_heads"] * case["rows"] * case["longest"] > 2 ** 31:
            continue
        return case


def _draw(rng):
    kind = rng.choice(["store", "fp8", "fp8", "exact", "exact", "rotate"])
    d = rng.choice([64, 128, 128, 128, 192, 256])
    kv = rng.choice([1, 2, 4, 8, 8, 16])
    per = rng.choice([1, 2, 4, 4, 5, 7, 8, 8, 16, 24])
    if kind == "rotate":
        return dict(kind=kind, rows=_between(rng, 1, 32768), q_heads=kv * per, kv_heads=kv, head_dim=d, rotary_dim=rng.choice([d, d, d // 2, 32]),
                    norm=rng.random() < 0.6, interleaved=rng.random() < 0.4, furthest=rng.choice([4096, 131072, 1 << 20]),
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    longest = _between(rng, 40, 131072)
    shortest = longest if rng.random() < 0.4 else max(1, longest // rng.choice([2, 8, 100]))
    rows = 1 if rng.random() < 0.4 else _between(rng, 2, min(longest, 8192))
    c = dict(kind=kind, seqs=_between(rng, 1, 128), shortest=shortest, longest=longest, rows=rows, kv_heads=kv, head_dim=d,
             dtype=rng.choice(["bf16", "bf16", "fp16"] + (["fp32"] if kind == "store" else [])))
    if kind == "store":
        return c
    windowed = kind == "exact" or rng.random() < 0.3
    c.update(q_heads=kv * per, window=_between(rng, 1, longest) if windowed else 0, sinks=rng.choice([0, 1, 4, 20]) if windowed else 0)
    return c


# ---- inputs -----------------------------------------------------------------------------------------------------------------

def _lengths(c):
    """The sequences' lengths, spread over the logarithm of shortest .. longest, odd ones among them."""
    n, lo, hi = c["seqs"], c["shortest"], c["longest"]
    if n == 1 or lo == hi:
        return [hi] * n
    return [int(round(lo * (hi / lo) ** (i / (n - 1)))) for i in range(n)]


def _runs(c):
    """The sequences' rows in the step."""
    return [min(n, c["rows"]) for n in _lengths(c)]


def _tails(c):
    """Tokens of the blocks that the step's rows go to."""
    return [n - (n - r) // PAGE * PAGE for n, r in zip(_lengths(c), _runs(c))]


def _scale_of(largest):
    """The exponent (int32) of the scale of a block whose largest finite value is `largest` (float32)."""
    mantissa, exponent = torch.frexp(largest)                          # largest = mantissa 2^exponent, 0.5 <= mantissa < 1; 448 = 0.875 2^9
    e = exponent - 9 + (mantissa > 0.875).to(torch.int32)
    return torch.where(largest == 0, torch.full_like(e, LOWEST), e.clamp(LOWEST, 119))


def _power(e, dt=torch.float32):
    """2^e exactly, of normal size (torch.ldexp and 2.0 ** e go by pow(), which is a step off here and there on a GPU, and
    16-bit values lie on the border between two of e4m3 often)."""
    return (e.to(torch.int32) + 127 << 23).view(torch.float32) if dt == torch.float32 else (e.long() + 1023 << 52).view(torch.float64)


def _to_f8(x, e):
    """x (float32) over 2^e, rounded to e4m3: what has no number of that size becomes the largest."""
    return (x * _power(-e)).clamp(-F8_MAX, F8_MAX).to(F8)


def _finite_size(x):
    return torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dt, H, d = DTYPES[c["dtype"]], c["kv_heads"], c["head_dim"]
    randn = lambda *shape: torch.randn(*shape, generator=g, device=DEVICE)
    if c["kind"] == "rotate":
        Hq, T, r = c["q_heads"], c["rows"], c["rotary_dim"]
        qkv = (randn(T, (Hq + 2 * H) * d) * torch.exp(0.5 * randn((Hq + 2 * H) * d))).to(dt)      # a projection's output
        s = dict(case=c, query=qkv[:, : Hq * d].view(T, Hq, d), key=qkv[:, Hq * d: (Hq + H) * d].view(T, H, d),
                 positions=torch.randint(c["furthest"], (T,), generator=g, device=DEVICE))
        s["inv_freq"] = 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64, device=DEVICE) / r)
        s["q_weight"], s["k_weight"] = ((1 + 0.2 * randn(d)).to(dt) if c["norm"] else None for _ in range(2))
        return s
    lens, runs = _lengths(c), _runs(c)
    B, pages = len(lens), [(n + PAGE - 1) // PAGE for n in lens]
    s = dict(case=c, max_len=max(lens), max_rows=max(runs), lens=torch.tensor(lens, dtype=torch.int32, device=DEVICE),
             starts=torch.tensor([0] + runs).cumsum(0).to(device=DEVICE, dtype=torch.int32))
    # the engine's cache, its blocks handed out in no order, a few of them to nobody
    blocks = sum(pages) + 3
    order = torch.randperm(blocks, generator=g, device=DEVICE).to(torch.int32)
    table = torch.zeros(B, max(pages), dtype=torch.int32, device=DEVICE)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at: at + n]
        at += n
    s["table"] = table
    # some channels of the keys are larger than others
    size = torch.exp(0.5 * randn(H, d))
    if c["kind"] == "exact":
        s["key_cache"], s["value_cache"] = (randn(blocks, PAGE, H, d) * size).to(dt), randn(blocks, PAGE, H, d).to(dt)
    else:
        for name, factor in (("key", size), ("value", torch.ones_like(size))):
            x = randn(blocks, PAGE, H, d) * factor
            e = _scale_of(x.abs().amax((1, 3)))
            s[name + "_cache"], s[name + "_scales"] = _to_f8(x, e[:, None, :, None]), (e + 127).to(torch.uint8)
            del x
    rows = sum(runs)
    if c["kind"] == "store":
        s["key"], s["value"] = (randn(rows, H, d) * size * 1.5).to(dt), randn(rows, H, d).to(dt)
        tails = _tails(c)
        s["tail_rows"], s["tails"] = sum(tails), torch.tensor([0] + tails).cumsum(0).to(device=DEVICE, dtype=torch.int32)
    else:
        s["query"] = randn(rows, c["q_heads"], d).to(dt)
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return {"store": _store, "fp8": _attend, "exact": _attend, "rotate": _rotate}[state["case"]["kind"]](state)


def _run_own(s):
    c = s["case"]
    if c["kind"] == "rotate":
        from turboquant_amd.rotary import rotate_heads
        q, k = rotate_heads(s["query"], s["key"], s["positions"], s["inv_freq"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=1e-6,
                            interleaved=c["interleaved"])
        return dict(query=q, key=k)
    if c["kind"] == "exact":
        from turboquant_amd.exact import ExactPagedCache
        cache = ExactPagedCache(s["key_cache"], s["value_cache"])
    else:
        from turboquant_amd.fp8 import Fp8PagedCache
        cache = Fp8PagedCache(s["key_cache"], s["value_cache"], s["key_scales"], s["value_scales"])
    if c["kind"] == "store":
        cache.write(s["key"], s["value"], s["starts"], s["table"], s["lens"])
        k, v = cache.read(s["tails"], s["table"], s["lens"], rows=s["tail_rows"], dtype=DTYPES[c["dtype"]])
        return _stored(s, k, v)
    seen = dict(window=c["window"] or None, sinks=c["sinks"], max_len=s["max_len"])
    if c["rows"] == 1:
        return cache.decode_attention(s["query"], s["table"], s["lens"], **seen)
    return cache.attention(s["query"], s["starts"], s["table"], s["lens"], max_rows=s["max_rows"], **seen)


def _stored(s, k, v):
    return dict(keys=k, values=v, key_cache=s["key_cache"], value_cache=s["value_cache"], key_scales=s["key_scales"],
                value_scales=s["value_scales"])


def _places(starts, rows, table, lens):
    """Of every row: its sequence, its token, the token's block and slot."""
    row = torch.arange(rows, device=starts.device)
    b = torch.searchsorted(starts[1:].long(), row, right=True)
    token = lens[b].long() - starts[b + 1] + row
    return b, token, table[b, token // PAGE].long(), token % PAGE


def _store(s):
    starts, table, lens = s["starts"].long(), s["table"], s["lens"]
    rows = s["key"].shape[0]
    b, token, block, slot = _places(starts, rows, table, lens)
    # a sequence's first block may hold earlier tokens
    first = lens.long() - (starts[1:] - starts[:-1])
    kept = first % PAGE
    head = table.gather(1, (first // PAGE).clamp_max(table.shape[1] - 1)[:, None])[:, 0].long()
    earlier = torch.arange(PAGE, device=lens.device) < kept[:, None]
    tb, _, tail_block, tail_slot = _places(s["tails"].long(), s["tail_rows"], table, lens)
    back = []
    for name in ("key", "value"):
        x, cache, scales = s[name].float(), s[name + "_cache"], s[name + "_scales"]
        e_old = scales[head].to(torch.int32) - 127
        held = cache.view(torch.uint8)[head].view(F8).float()
        largest = torch.zeros(scales.shape, device=x.device)
        largest.scatter_reduce_(0, block[:, None].expand(-1, x.shape[1]), _finite_size(x).amax(-1), "amax")
        e = _scale_of(largest)
        e[head] = torch.where((kept > 0)[:, None], torch.maximum(e[head], e_old), e[head])
        # earlier tokens, rounded again where their scale has grown
        again = _to_f8(held, (e[head] - e_old)[:, None, :, None])
        hb, hs = earlier.nonzero(as_tuple=True)
        raw = cache.view(torch.uint8)
        raw[head[hb], hs] = again.view(torch.uint8)[hb, hs]
        raw[block, slot] = _to_f8(x, e[block][:, :, None]).view(torch.uint8)
        scales[block] = (e[block] + 127).to(torch.uint8)
        back.append(_values(cache, scales, tail_block, tail_slot).to(s[name].dtype))
    return _stored(s, *back)


def _values(cache, scales, block, slot):
    """Tokens at (block, slot) of the 8-bit cache in 32 bits."""
    q = cache.view(torch.uint8)[block, slot].view(F8).float()
    return q * _power(scales[block].to(torch.int32)[..., None] - 127)


def _attend(s):
    c, lens, table, starts = s["case"], s["lens"].long(), s["table"], s["starts"].long()
    B, H, d, R, q = c["seqs"], c["kv_heads"], c["head_dim"], s["max_rows"], s["query"]
    run = starts[1:] - starts[:-1]
    # the tokens that any row sees: with a window the newest ones and the first few, in front of them
    longest, window, sinks = s["max_len"], c["window"], c["sinks"]
    newest = longest if not window else min(longest, window + R - 1)
    front = min(sinks, longest) if newest < longest else 0
    token = torch.cat([torch.arange(front, device=q.device).expand(B, front),
                       (lens[:, None] - newest + torch.arange(newest, device=q.device))], 1)
    there = token >= 0
    there[:, :front] = token[:, :front] < (lens - newest)[:, None]
    token = token.clamp_min(0)
    block, slot = table.gather(1, token // PAGE).long(), token % PAGE

    def rows_of(name):                                                  # (B, H, 1, tokens, d) in 32 bits
        cache = s[name + "_cache"]
        x = _values(cache, s[name + "_scales"], block, slot) if c["kind"] == "fp8" else cache[block, slot].float()
        return x.transpose(1, 2).contiguous()

    # rows of every sequence side by side, the first ones empty where it has fewer
    row = starts[1:, None] - R + torch.arange(R, device=q.device)
    mine = row >= starts[:-1, None]
    x = q[row.clamp_min(0)].float() * mine[:, :, None, None]            # (B, R, Hq, d)
    G = c["q_heads"] // H
    x = x.view(B, R, H, G, d).permute(0, 2, 3, 1, 4).reshape(B, H, G * R, d)
    scores = (x @ rows_of("key").transpose(-1, -2)).view(B, H, G, R, -1)
    scores *= 1 / math.sqrt(d)
    at = (lens[:, None] - R + torch.arange(R, device=q.device))[:, :, None]                     # a row's token
    t = token[:, None, :]
    visible = (t <= at) & there[:, None, :]
    if window:
        visible &= (t > at - window) | (t < sinks)
    scores.masked_fill_(~visible[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores -= torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = scores.exp_()
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total == 0, torch.ones_like(total), total)
    out = p.view(B, H, G * R, -1) @ rows_of("value")
    out = out.view(B, H, G, R, d).permute(0, 3, 1, 2, 4).reshape(B, R, H * G, d)
    return out[mine].to(q.dtype)


def _rotate(s):
    c = s["case"]
    half = c["rotary_dim"] // 2
    angle = s["positions"].double()[:, None] * s["inv_freq"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    got = {}
    for name, weight in (("query", s["q_weight"]), ("key", s["k_weight"])):
        x = s[name].float()
        if c["norm"]:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.float()
        r = x[..., : 2 * half]
        a, b = (r[..., 0::2], r[..., 1::2]) if c["interleaved"] else (r[..., :half], r[..., half:])
        a, b = a * cos - b * sin, b * cos + a * sin
        r = torch.stack([a, b], -1).flatten(-2) if c["interleaved"] else torch.cat([a, b], -1)
        got[name] = torch.cat([r, x[..., 2 * half:]], -1).to(s[name].dtype)
    return got


# ---- what a pass cannot do without --------------------------------------------------------------------------------------------

def _seen(c, n, p):
    """Tokens that the row at position p sees."""
    if not c["window"] or p + 1 <= c["window"]:
        return p + 1
    return c["window"] + min(c["sinks"], p + 1 - c["window"])


def work(case):
    c, size, H, d = case, 4 if case["dtype"] == "fp32" else 2, case["kv_heads"], case["head_dim"]
    if c["kind"] == "rotate":
        n = c["rows"] * (c["q_heads"] + H) * d
        return {"bytes": 2 * n * size + 8 * c["rows"], "flops": 8 * n}
    lens, runs = _lengths(c), _runs(c)
    table = 8 * len(lens)
    if c["kind"] == "store":
        written, back = sum(runs) * H * d, sum(_tails(c)) * H * d
        blocks = sum((n + PAGE - 1) // PAGE - (n - r) // PAGE for n, r in zip(lens, runs))
        return {"bytes": 2 * (written * (size + 1) + back * (size + 1) + 2 * blocks * H) + table + 8 * blocks, "flops": 4 * written + 2 * back}
    read = pairs = blocks = 0
    for n, r in zip(lens, runs):
        # the tokens that any row sees, and the pairs of a row and a token
        low = n - r
        tokens = n if not c["window"] else min(n, c["window"] + r - 1)
        tokens += min(c["sinks"], n - tokens)
        read += tokens
        blocks += (tokens + PAGE - 1) // PAGE
        if not c["window"]:
            pairs += r * low + r * (r + 1) // 2
        else:
            pairs += sum(_seen(c, n, p) for p in range(low, n))
    held = size if c["kind"] == "exact" else 1
    scales = 0 if c["kind"] == "exact" else 2 * blocks * H
    return {"bytes": 2 * read * H * d * held + scales + 2 * sum(runs) * c["q_heads"] * d * size + table + 4 * blocks,
            "flops": 4 * pairs * c["q_heads"] * d}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("fp8", "exact") and work(case)["flops"] > 4e12:
        return None
    return {"store": _exact_store, "fp8": _exact_attend, "exact": _exact_attend, "rotate": _exact_rotate}[case["kind"]](s)


def _round_e4m3(x):
    """x (float64) to the nearest number of e4m3, ties to the even one."""
    step = _power((torch.frexp(x)[1] - 1).clamp_min(-6) - 3, torch.float64)
    return torch.round(x / step) * step


def _exact_store(s):
    c, starts = s["case"], s["starts"].tolist()
    out = {}
    for name in ("key", "value"):
        got = []
        for b, (n, run, tail) in enumerate(zip(_lengths(c), _runs(c), _tails(c))):
            at = torch.arange(n - tail, n, device=DEVICE)
            block, slot, kept = s["table"][b, at // PAGE].long(), at % PAGE, tail - run
            new = s[name][starts[b]: starts[b + 1]].double()
            old = s[name + "_cache"][block[:kept], slot[:kept]].double() * _power(s[name + "_scales"][block[:kept]].long() - 127, torch.float64)[..., None]
            e_old = (s[name + "_scales"][block[:1]].double() - 127) if kept else torch.full((1, c["kv_heads"]), float(LOWEST), device=DEVICE)
            whole = torch.cat([torch.zeros_like(old), new])
            pages = torch.nn.functional.pad(whole, (0, 0, 0, 0, 0, -tail % PAGE)).unflatten(0, (-1, PAGE))
            largest = pages.abs().amax((1, 3))
            # the least power of two that brings the largest value to 448 at most
            e = torch.full_like(largest, float(LOWEST))
            e[largest > 0] = torch.ceil(torch.log2(largest[largest > 0] / 448))
            size = _power(e, torch.float64)
            e = torch.where(largest > 448 * size, e + 1, torch.where((largest <= 224 * size) & (largest > 0), e - 1, e)).clamp_min(LOWEST)
            e[:1] = torch.maximum(e[:1], e_old)
            factor = _power(e, torch.float64)[torch.arange(tail, device=DEVICE) // PAGE][..., None]
            x = torch.cat([old, new]) / factor
            got.append(_round_e4m3(x) * factor)
        out[name + "s"] = torch.cat(got)
    return dict(keys=out["keys"], values=out["values"], key_cache=None, value_cache=None, key_scales=None, value_scales=None)


def _exact_attend(s):
    c, starts = s["case"], s["starts"].tolist()
    G, d, q = c["q_heads"] // c["kv_heads"], c["head_dim"], s["query"].double()
    out = torch.zeros_like(q)

    def tokens(name, at, b, h):
        block, slot = s["table"][b, at // PAGE].long(), at % PAGE
        x = s[name + "_cache"][block, slot, h].double()
        return x * _power(s[name + "_scales"][block, h].long() - 127, torch.float64)[:, None] if c["kind"] == "fp8" else x

    for b, n in enumerate(_lengths(c)):
        run = starts[b + 1] - starts[b]
        at = torch.arange(n, device=DEVICE)
        p = torch.arange(n - run, n, device=DEVICE)[:, None]
        hidden = at > p
        if c["window"]:
            at = at[(at < c["sinks"]) | (at > n - run - c["window"])]
            hidden = (at > p) | ((at <= p - c["window"]) & (at >= c["sinks"]))
        for h in range(c["kv_heads"]):
            k, v = tokens("key", at, b, h), tokens("value", at, b, h)
            for head in range(h * G, (h + 1) * G):
                x = (q[starts[b]: starts[b + 1], head] @ k.T / d ** 0.5).masked_fill(hidden, -math.inf)
                out[starts[b]: starts[b + 1], head] = torch.softmax(x, -1) @ v
    return out


def _exact_rotate(s):
    c, half = s["case"], s["case"]["rotary_dim"] // 2
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEVICE), s["positions"].double()[:, None] * s["inv_freq"])[:, None]
    got = {}
    for name, weight in (("query", s["q_weight"]), ("key", s["k_weight"])):
        x = s[name].double()
        if c["norm"]:
            x = x / ((x ** 2).mean(-1, keepdim=True) + 1e-6).sqrt() * weight.double()
        first = torch.arange(half, device=DEVICE) * (2 if c["interleaved"] else 1)
        second = first + (1 if c["interleaved"] else half)
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        got[name] = x
    return got
