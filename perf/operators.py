"""The exact paged cache's operators as timed cases: decode attention, the weights of a prompt's window, eviction by weight.

A serving engine holds keys and values as (blocks, 16, KV heads, head_dim) tensors that sequences reach through block tables.
A case is a dict of plain values; `kind` says which operator it takes:

  decode  attention of one new token per sequence over that cache, with or without every token's attention weight added to
          a running sum per KV head (`ExactPagedCache.decode_attention`)
  window  the weight that the newest queries of every prompt give to every token of the cache, added to the same sums: what
          a cache knows about a prompt before the first token is decoded (`ExactPagedCache.add_window_weights`)
  evict   choose the tokens that stay by those sums, move them together and shorten the sequences (`select_evictions`,
          `ExactPagedCache.move_tokens`)

With `own` false the same is computed by elementary torch operations in 32 bits.
"""

import math

import torch

own = False

PAGE = 16
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEVICE = "cuda:0"


def listed():
    return [
        # ---- one new token per sequence ------------------------------------------------------------------------------------
        # a chat's reply, one sequence in one layer: launches and latency are what counts
        dict(name="decode_chat", kind="decode", seqs=1, shortest=700, longest=700, q_heads=32, kv_heads=8, head_dim=128,
             weights=False, dtype="bf16"),
        # a batch of chats of a grouped-query model whose cache is to be cut by weight
        dict(name="decode_batch", kind="decode", seqs=16, shortest=8192, longest=8192, q_heads=32, kv_heads=8, head_dim=128,
             weights=True, dtype="bf16"),
        # one long document, wide heads, few of them
        dict(name="decode_long", kind="decode", seqs=1, shortest=131072, longest=131072, q_heads=16, kv_heads=2,
             head_dim=256, weights=True, dtype="bf16"),
        # many requests of very different length, an odd number of heads per KV head
        dict(name="decode_ragged", kind="decode", seqs=96, shortest=61, longest=8190, q_heads=40, kv_heads=8, head_dim=128,
             weights=True, dtype="fp16"),
        # latent attention: every query head on one KV head of 576
        dict(name="decode_latent", kind="decode", seqs=16, shortest=8192, longest=8192, q_heads=128, kv_heads=1,
             head_dim=576, weights=False, dtype="bf16"),
        # multi-head attention of an unquantised model
        dict(name="decode_fp32", kind="decode", seqs=8, shortest=1500, longest=2048, q_heads=16, kv_heads=16, head_dim=64,
             weights=True, dtype="fp32"),
        # ---- the newest queries of a prompt --------------------------------------------------------------------------------
        # the prompt of a chat
        dict(name="window_chat", kind="window", seqs=1, shortest=1500, longest=1500, window=32, q_heads=32, kv_heads=8,
             head_dim=128, dtype="bf16"),
        # documents, all of their layer's heads
        dict(name="window_documents", kind="window", seqs=4, shortest=32768, longest=32768, window=32, q_heads=32, kv_heads=8,
             head_dim=128, dtype="bf16"),
        # a prefill step of several prompts of odd lengths, some shorter than the window, wide heads
        dict(name="window_ragged", kind="window", seqs=9, shortest=17, longest=4099, window=64, q_heads=16, kv_heads=2,
             head_dim=256, dtype="fp16"),
        # ---- eviction ------------------------------------------------------------------------------------------------------
        # a full decode batch at its budget, cut back every 16 tokens
        dict(name="evict_step", kind="evict", seqs=32, shortest=2064, longest=2064, budget=2048, sinks=4, recent=256,
             kv_heads=8, head_dim=128, again=True, dtype="bf16"),
        # prompts of documents, cut to an eighth
        dict(name="evict_documents", kind="evict", seqs=4, shortest=32768, longest=32768, budget=4096, sinks=4, recent=512,
             kv_heads=8, head_dim=128, again=False, dtype="bf16"),
        # one long document, wide heads, few of them: rows too long for one compute unit
        dict(name="evict_long", kind="evict", seqs=1, shortest=131072, longest=131072, budget=16384, sinks=16, recent=1024,
             kv_heads=2, head_dim=256, again=False, dtype="bf16"),
    ]


# ---- drawn cases ----------------------------------------------------------------------------------------------------------

def _between(rng, lo, hi):
    """A whole number spread over the logarithm of lo .. hi."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the same ranges, no more work than the largest listed ones."""
    most = [work(c) for c in listed()]
    while True:
        case = _draw(rng)
        w = work(case)
        if all(w[k] <= max(m[k] for m in most) for k in ("bytes", "flops")) and w["bytes"] > 1e5:
            return case


def _draw(rng):
    kind = rng.choice(["decode", "decode", "window", "evict"])
    d = rng.choice([64, 128, 128, 128, 192, 256, 512, 576])
    kv = 1 if d > 256 else rng.choice([1, 2, 4, 8, 8, 16])
    per = rng.choice([8, 16, 32, 64, 128]) if d > 256 else rng.choice([1, 2, 4, 4, 5, 7, 8, 8, 16, 24])
    longest = _between(rng, 40, 131072)
    shortest = longest if rng.random() < 0.4 else max(1, longest // rng.choice([2, 8, 100]))
    c = dict(kind=kind, seqs=_between(rng, 1, 128), shortest=shortest, longest=longest, kv_heads=kv, head_dim=d,
             dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    if kind == "evict":
        budget = _between(rng, 24, longest)
        sinks, recent = rng.choice([0, 1, 4, 16]), rng.choice([0, budget // 8, budget // 2])
        c.update(budget=budget, sinks=min(sinks, budget - recent), recent=recent, again=rng.random() < 0.5)
        return c
    c["q_heads"] = kv * per
    if kind == "window":
        c["window"] = _between(rng, 1, 64)
    else:
        c["weights"] = rng.random() < 0.5
    return c


# ---- inputs -----------------------------------------------------------------------------------------------------------------

def _lengths(c):
    """The sequences' lengths, spread over the logarithm of shortest .. longest, odd ones among them."""
    n, lo, hi = c["seqs"], c["shortest"], c["longest"]
    if n == 1 or lo == hi:
        return [hi] * n
    return [int(round(lo * (hi / lo) ** (i / (n - 1)))) for i in range(n)]


def _seen(c, length):
    """Tokens that a sequence has had: more than it holds where its cache has been cut before."""
    return 2 * length if c.get("again") else length


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dt, H, d, B = DTYPES[c["dtype"]], c["kv_heads"], c["head_dim"], c["seqs"]
    lens = _lengths(c)
    pages = [(n + PAGE - 1) // PAGE for n in lens]
    width = max(pages)
    randn = lambda *shape: torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32 if dt == torch.float32 else dt)
    s = dict(case=c, max_len=max(lens), lens=torch.tensor(lens, dtype=torch.int32, device=DEVICE))
    # the engine's cache, its blocks handed out in no order, a few of them to nobody
    blocks = sum(pages) + 3
    order = torch.randperm(blocks, generator=g, device=DEVICE).to(torch.int32)
    table = torch.zeros(B, width, dtype=torch.int32, device=DEVICE)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at: at + n]
        at += n
    s.update(table=table, keys=randn(blocks, PAGE, H, d), values=randn(blocks, PAGE, H, d))
    if c["kind"] == "decode":
        s["query"] = randn(B, c["q_heads"], d) * 2
        # sums over a few steps before this one
        s["weights"] = torch.rand(B, H, s["max_len"], generator=g, device=DEVICE) * (8 / max(lens)) if c["weights"] else None
    elif c["kind"] == "window":
        rows = [min(n, c["window"]) for n in lens]
        starts = torch.tensor([0] + rows).cumsum(0)
        s["query"] = randn(int(starts[-1]), c["q_heads"], d) * 2
        s["starts"] = starts.to(device=DEVICE, dtype=torch.int32)
        s["weights"] = torch.zeros(B, H, s["max_len"], device=DEVICE)
    else:
        # sums of probabilities: a few tokens have most of them, some have none
        L = s["max_len"]
        w = torch.exp(2 * torch.randn(B, H, L, generator=g, device=DEVICE))
        w[torch.rand(B, H, L, generator=g, device=DEVICE) < 0.05] = 0
        inside = torch.arange(L, device=DEVICE) < s["lens"][:, None, None]
        s["weights"] = w * inside
        s["seen"] = torch.tensor([_seen(c, n) for n in lens], dtype=torch.int32, device=DEVICE)
        pos = torch.arange(L, dtype=torch.int32, device=DEVICE).expand(B, H, L).clone()
        if c["again"]:
            # what an earlier cut left of the older tokens lies in no order before the newest of them
            for b, n in enumerate(lens):
                new = min(n, PAGE)
                old = torch.rand(H, 2 * n - new, generator=g, device=DEVICE).argsort(-1)[:, : n - new]
                pos[b, :, : n - new] = old.to(torch.int32)
                pos[b, :, n - new:] = 2 * n - new + torch.arange(L - n + new, dtype=torch.int32, device=DEVICE)
        s["positions"] = pos
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return {"decode": _decode, "window": _window, "evict": _evict}[state["case"]["kind"]](state)


def _run_own(s):
    from turboquant_amd.eviction import select_evictions
    from turboquant_amd.exact import ExactPagedCache
    c, cache = s["case"], ExactPagedCache(s["keys"], s["values"])
    if c["kind"] == "decode":
        out = cache.decode_attention(s["query"], s["table"], s["lens"], weights=s["weights"], max_len=s["max_len"])
        return dict(out=out, weights=s["weights"])
    if c["kind"] == "window":
        cache.add_window_weights(s["query"], s["starts"], s["table"], s["lens"], s["weights"], window=c["window"],
                                 max_len=s["max_len"])
        return s["weights"]
    e = select_evictions(s["weights"], s["positions"], s["lens"], c["budget"], seen=s["seen"], sinks=c["sinks"],
                         recent=c["recent"])
    cache.move_tokens(e, s["table"])
    return dict(lens=e.lens, count=e.count, dst=e.dst, src=e.src, weights=e.weights, positions=e.positions, keys=s["keys"],
                values=s["values"])


def _rows(cache, table, L):
    """Every sequence's tokens (B, H, L, d) in 32 bits."""
    B = table.shape[0]
    t = cache[table.long()].float()                                        # (B, pages, 16, H, d)
    return t.reshape(B, -1, *cache.shape[2:])[:, :L].transpose(1, 2).contiguous()


def _probabilities(scores):
    """softmax over the last dimension; a row of nothing but -inf has no weight anywhere."""
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _decode(s):
    c, L, q = s["case"], s["max_len"], s["query"]
    B, H, d = c["seqs"], c["kv_heads"], c["head_dim"]
    k = _rows(s["keys"], s["table"], L)
    scores = q.float().view(B, H, -1, d) @ k.transpose(-1, -2) / math.sqrt(d)        # (B, H, heads on one, L)
    del k
    beyond = torch.arange(L, device=q.device) >= s["lens"][:, None, None, None]
    p = _probabilities(scores.masked_fill(beyond, -math.inf))
    out = (p @ _rows(s["values"], s["table"], L)).view(B, -1, d).to(q.dtype)
    if s["weights"] is not None:
        s["weights"] += p.sum(2)
    return dict(out=out, weights=s["weights"])


def _window(s):
    c, L, W = s["case"], s["max_len"], s["case"]["window"]
    B, H, d = c["seqs"], c["kv_heads"], c["head_dim"]
    starts, lens = s["starts"].long(), s["lens"].long()
    # the newest W rows of every sequence, from the back; those before its first are of no sequence
    back = torch.arange(W, device=lens.device)
    row = starts[1:, None] - 1 - back
    there = row >= starts[:-1, None]
    q = s["query"][row.clamp_min(0)].float() * there[:, :, None, None]                # (B, W, Hq, d)
    q = q.view(B, W, H, -1, d).permute(0, 2, 3, 1, 4).reshape(B, H, -1, d)
    scores = (q @ _rows(s["keys"], s["table"], L).transpose(-1, -2) / math.sqrt(d)).view(B, H, -1, W, L)
    last = (lens[:, None] - 1 - back)[:, None, None, :, None]
    hidden = (torch.arange(L, device=lens.device) > last) | ~there[:, None, None, :, None]
    s["weights"] += _probabilities(scores.masked_fill(hidden, -math.inf)).sum((2, 3))
    return s["weights"]


def _evict(s):
    c, w, pos = s["case"], s["weights"], s["positions"]
    B, H, L = w.shape
    budget, most = c["budget"], max(1, min(c["budget"], L - c["budget"]))
    lens, seen = s["lens"].long()[:, None, None], s["seen"].long()[:, None, None]
    slot = torch.arange(L, device=w.device).expand(B, H, L)
    inside = slot < lens
    # the order of who stays: sinks and newest tokens, then by weight (one that is no number last), the lower slot of two alike
    value = torch.where(torch.isnan(w), torch.full_like(w, -math.inf), w).clamp_max(torch.finfo(torch.float32).max)
    held = (pos < c["sinks"]) | (pos >= seen - c["recent"])
    value = value.masked_fill(held, math.inf)
    by = value.sort(dim=-1, descending=True, stable=True).indices
    by = by.gather(-1, inside.gather(-1, by).to(torch.uint8).sort(dim=-1, descending=True, stable=True).indices)
    rank = torch.empty_like(by).scatter_(-1, by, slot)
    stays = inside & ((rank < budget) | (lens <= budget))
    hole, mover = inside & ~stays & (slot < budget), stays & (slot >= budget)
    count = mover.sum(-1)
    # the n-th hole takes the n-th of those that stay behind the budget
    nth = torch.arange(most, device=w.device).expand(B, H, most)
    found = nth < count[..., None]

    def list_of(mask):
        first = mask.to(torch.uint8).sort(dim=-1, descending=True, stable=True).indices[..., :most]
        return torch.where(found, first, torch.full_like(first, -1))

    dst, src = list_of(hole), list_of(mover)
    b, h, n = found.nonzero(as_tuple=True)
    to, of = dst[b, h, n], src[b, h, n]
    left = torch.where(lens > budget, torch.full_like(lens, budget), lens)
    weights, positions = w.clone(), pos.clone()
    weights[b, h, to], positions[b, h, to] = w[b, h, of], pos[b, h, of]
    vacant = slot >= left
    weights.masked_fill_(vacant, 0)
    positions = torch.where(vacant, (seen + slot - left).to(torch.int32), positions)
    table = s["table"].long()
    to_block, of_block = table[b, to // PAGE], table[b, of // PAGE]
    for cache in (s["keys"], s["values"]):
        cache[to_block, to % PAGE, h] = cache[of_block, of % PAGE, h]
    return dict(lens=left.view(B).to(torch.int32), count=count.to(torch.int32), dst=dst.to(torch.int32), src=src.to(torch.int32),
                weights=weights, positions=positions, keys=s["keys"], values=s["values"])


# ---- what a pass cannot do without --------------------------------------------------------------------------------------------

def work(case):
    c, size = case, 4 if case["dtype"] == "fp32" else 2
    H, d, lens = c["kv_heads"], c["head_dim"], _lengths(case)
    tokens, L = sum(lens), max(lens)
    table = 4 * sum((n + PAGE - 1) // PAGE for n in lens) + 4 * len(lens)
    if c["kind"] == "decode":
        rows = c["seqs"] * c["q_heads"] * d * size
        return {"bytes": 2 * tokens * H * d * size + 2 * rows + table + (8 * tokens * H if c["weights"] else 0),
                "flops": 4 * tokens * c["q_heads"] * d}
    if c["kind"] == "window":
        rows = [min(n, c["window"]) for n in lens]
        return {"bytes": tokens * H * d * size + sum(rows) * c["q_heads"] * d * size + 8 * tokens * H + table,
                "flops": 2 * c["q_heads"] * d * sum(r * n - r * (r - 1) // 2 for r, n in zip(rows, lens))}
    # the tokens that move, if weight says nothing about age: the newest, and the others' share behind the budget
    moved = 0.0
    for n in lens:
        if n > c["budget"]:
            others = n - c["sinks"] - c["recent"]
            behind = max(0, n - c["recent"] - c["budget"])
            kept = c["budget"] - c["sinks"] - c["recent"]
            moved += min(c["recent"], n - c["budget"]) + kept * behind / max(1, others)
    return {"bytes": H * moved * (4 * d * size + 8) + 8 * H * (tokens + len(lens) * L) + table, "flops": H * tokens}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"decode": _exact_decode, "window": _exact_window, "evict": _exact_evict}[case["kind"]](s)


def _sequence(cache, table, b, n, h):
    """Tokens 0 .. n - 1 of sequence b at KV head h, in 64 bits."""
    at = torch.arange(n, device=table.device)
    return cache[table[b, at // PAGE].long(), at % PAGE, h].double()


def _exact_decode(s):
    c, q = s["case"], s["query"].double()
    per, d = c["q_heads"] // c["kv_heads"], c["head_dim"]
    out = torch.zeros_like(q)
    weights = None if s["weights"] is None else s["weights"].double()
    for b, n in enumerate(_lengths(c)):
        for h in range(c["kv_heads"]):
            heads = slice(h * per, (h + 1) * per)
            p = torch.softmax(q[b, heads] @ _sequence(s["keys"], s["table"], b, n, h).T / d ** 0.5, -1)
            out[b, heads] = p @ _sequence(s["values"], s["table"], b, n, h)
            if weights is not None:
                weights[b, h, :n] += p.sum(0)
    return dict(out=out, weights=weights)


def _exact_window(s):
    c, weights = s["case"], s["weights"].double()
    per, d = c["q_heads"] // c["kv_heads"], c["head_dim"]
    starts = s["starts"].tolist()
    for b, n in enumerate(_lengths(c)):
        r = min(c["window"], starts[b + 1] - starts[b])
        q = s["query"][starts[b + 1] - r: starts[b + 1]].double()
        unseen = torch.ones(r, n, dtype=torch.bool, device=q.device).triu(n - r + 1)
        for h in range(c["kv_heads"]):
            k = _sequence(s["keys"], s["table"], b, n, h)
            for head in range(h * per, (h + 1) * per):
                weights[b, h, :n] += torch.softmax((q[:, head] @ k.T / d ** 0.5).masked_fill(unseen, -math.inf), -1).sum(0)
    return weights


def _exact_evict(s):
    c, lens, seen = s["case"], _lengths(s["case"]), s["seen"].tolist()
    weights, positions = s["weights"].double(), s["positions"].clone()
    keys, values, table = s["keys"].double(), s["values"].double(), s["table"]
    for b, n in enumerate(lens):
        if n <= c["budget"]:
            weights[b, :, n:] = 0
            continue
        for h in range(c["kv_heads"]):
            w, p = s["weights"][b, h, :n].double(), s["positions"][b, h, :n]
            w = w.masked_fill((p < c["sinks"]) | (p >= seen[b] - c["recent"]), math.inf)
            kept = torch.zeros(n, dtype=torch.bool, device=w.device)
            kept[torch.argsort(-w, stable=True)[: c["budget"]]] = True
            to, of = (~kept[: c["budget"]]).nonzero()[:, 0], c["budget"] + kept[c["budget"]:].nonzero()[:, 0]
            weights[b, h, to] = s["weights"][b, h, of].double()
            weights[b, h, c["budget"]:] = 0
            for new, old in ((keys, s["keys"]), (values, s["values"])):
                new[table[b, to // PAGE].long(), to % PAGE, h] = old[table[b, of // PAGE].long(), of % PAGE, h].double()
    return dict(lens=None, count=None, dst=None, src=None, weights=weights, positions=None, keys=keys, values=values)
