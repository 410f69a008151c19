"""A step's keys and values into the 8-bit cache and back, against the definition in 64 bits: every number equal."""

import pytest
import torch

from tests.step_helpers import DTYPES, F8, LOWEST, PAGE, Blocks8, Step, e4m3
from turboquant_amd.fp8 import Fp8PagedCache

pytestmark = pytest.mark.gpu


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0))


class Writer:
    """Sequences written step by step, here and by the definition."""

    def __init__(self, gpu, pages, H, d, seed=0, garbage=True):
        g = torch.Generator().manual_seed(seed)
        self.gpu, self.H, self.d, self.blocks = gpu, H, d, sum(pages) + 2
        order = torch.randperm(self.blocks, generator=g).to(torch.int32)
        self.table = torch.full((len(pages), max(pages)), -1, dtype=torch.int32)
        at = 0
        for b, p in enumerate(pages):
            self.table[b, :p] = order[at: at + p]
            at += p
        self.cache = Fp8PagedCache.allocate(self.blocks, H, d, gpu)
        if garbage:                                            # of the sequences that had these blocks before
            for t in (self.cache.key_cache, self.cache.value_cache):
                t.view(torch.uint8).random_(0, 256)
            for t in (self.cache.key_scales, self.cache.value_scales):
                t.random_(0, 256)
        self.want = Blocks8(self.blocks, H, d), Blocks8(self.blocks, H, d)
        self.len = [0] * len(pages)

    def step(self, runs, k, v, extra=0):
        """k, v on the CPU."""
        starts = torch.tensor([0] + list(runs)).cumsum(0)
        self.len = [n + r for n, r in zip(self.len, runs)]
        self.cache.write(k.to(self.gpu), v.to(self.gpu), starts.to(self.gpu), self.table.to(self.gpu), torch.tensor(self.len, device=self.gpu))
        for x, want in ((k, self.want[0]), (v, self.want[1])):
            for b, r in enumerate(runs):
                n, t = self.len[b], self.len[b] - r
                while t < n:
                    end = min(n, (t // PAGE + 1) * PAGE)
                    row = int(starts[b]) + t - (n - r)
                    want.write(x[row: row + end - t], int(self.table[b, t // PAGE]), t % PAGE)
                    t = end

    def check(self, dtype=torch.float32):
        starts = torch.tensor([0] + self.len).cumsum(0)
        got = self.cache.read(starts.to(self.gpu), self.table.to(self.gpu), torch.tensor(self.len, device=self.gpu), rows=int(starts[-1]), dtype=dtype)
        for x, want, scales in zip(got, self.want, (self.cache.key_scales, self.cache.value_scales)):
            values = want.values()
            for b, n in enumerate(self.len):
                t = torch.arange(n)
                block = self.table[b, t // PAGE].long()
                assert torch.equal(scales.cpu()[block].double() - 127, want.e[block]), f"scales of sequence {b}"
                assert same(x[starts[b]: starts[b + 1]].cpu(), values[block, t % PAGE].to(dtype)), f"sequence {b}"
        return got


@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_prompts_then_tokens(gpu, dtype, d):
    w = Writer(gpu, [4, 1, 6, 2, 3], 3, d)
    g = torch.Generator().manual_seed(d)
    # prompts (none of one sequence), a chunk that goes on inside a block, tokens, some of them much larger than those before
    for runs, size in (([37, 1, 80, 0, 16], 1.0), ([3, 0, 7, 17, 1], 0.3), ([1, 1, 1, 1, 1], 40.0), ([1, 1, 0, 1, 1], 1e-3), ([1, 1, 1, 1, 1], 1.0)):
        k, v = (size * torch.randn(sum(runs), 3, d, generator=g) * torch.exp(torch.randn(1, 3, 1, generator=g)) for _ in range(2))
        w.step(runs, k.to(DTYPES[dtype]), v.to(DTYPES[dtype]))
        w.check(DTYPES[dtype])


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_every_kind_of_value(gpu, dtype):
    """Zeros, the type's smallest and largest numbers, infinities, NaN, a block of nothing else; borders between two numbers of e4m3."""
    dt = DTYPES[dtype]
    info = torch.finfo(dt)
    w = Writer(gpu, [1] * 8, 1, 64)
    x = torch.randn(8 * PAGE, 1, 64, generator=torch.Generator().manual_seed(1))
    x[:16] = 0
    x[16:32] = torch.randn(16, 1, 64) * info.tiny
    x[32:48] *= float(info.max) / 8
    x[48] = float("inf")
    x[50, 0, 3], x[51, 0, 4], x[52, 0, 5] = float("inf"), -float("inf"), float("nan")
    x[64:80] = float("nan")
    x[80:96] = -float("inf")
    grid = torch.arange(-512, 512).view(16, 1, 64) / 1.0                      # ties: every half step between numbers of e4m3 below 512
    x[96:112] = grid.clamp(-448, 448)
    x[112:] = grid / 4096 * 2.0 ** -9
    x[112, 0, 0] = 448.0
    w.step([16] * 8, x.to(dt), (-x).to(dt))
    w.check()


def test_powers_of_two_and_their_neighbours(gpu):
    """A block's largest value at 448 2^i, just below and just above: the scale steps there and nowhere else."""
    at = [2.0 ** i for i in (-117, -100, -20, -1, 0, 1, 30, 110)]
    largest = torch.tensor([y for s in at for y in (448 * s, 448 * s * (1 - 2.0 ** -23), 448 * s * (1 + 2.0 ** -23), 224 * s, 225 * s)])
    w = Writer(gpu, [1] * len(largest), 1, 64)
    x = torch.randn(16 * len(largest), 1, 64, generator=torch.Generator().manual_seed(2))
    x = x.clamp(-1, 1) * largest.repeat_interleave(16)[:, None, None] * 0.9
    x[::16, 0, 7] = largest
    w.step([16] * len(largest), x, -x)
    w.check()


@pytest.mark.parametrize("view", ["heads apart", "tokens apart", "columns", "odd", "negated", "heads first"])
def test_inputs_of_other_layouts(gpu, view):
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(21, 2, 64, generator=g).bfloat16() for _ in range(2))
    w, plain = Writer(gpu, [2, 1], 2, 64), Writer(gpu, [2, 1], 2, 64)

    def as_view(x):
        x = x.to(gpu)
        if view == "heads apart":
            return torch.cat([x, x], -1)[..., :64]
        if view == "tokens apart":
            return torch.cat([x, x], 1)[:, :2]
        if view == "columns":
            return torch.cat([x.flatten(1)] * 3, 1)[:, 128:256].view(21, 2, 64)
        if view == "odd":
            return torch.cat([x.flatten()[:3], x.flatten()])[3:].view(21, 2, 64)
        if view == "negated":
            return torch._neg_view(-x)
        return x.transpose(0, 1).contiguous().transpose(0, 1)
    starts, lens = torch.tensor([0, 20, 21], device=gpu), torch.tensor([20, 1], device=gpu)
    w.cache.write(as_view(k), as_view(v), starts, w.table.to(gpu), lens)
    plain.step([20, 1], k, v)
    plain.check()
    w.len, w.want = plain.len, plain.want
    w.check()


def test_what_has_no_place_is_left_out(gpu):
    """Rows in front of token 0, behind the table, in blocks outside the cache, of no sequence: nothing is written for them, nothing else is lost."""
    H, d = 2, 64
    cache = Fp8PagedCache.allocate(6, H, d, gpu)
    for t in cache.tensors().values():
        t.view(torch.uint8).fill_(17)
    k, v = (torch.randn(60, H, d, generator=torch.Generator().manual_seed(4)) for _ in range(2))
    # 0: more rows than tokens; 1: longer than its table; 2: a block outside; 3: no tokens and no rows; 4: a negative length
    table = torch.tensor([[0, -1], [1, 2], [9, 3], [4, 4], [5, 5]], dtype=torch.int32, device=gpu)
    starts = torch.tensor([0, 7, 17, 37, 37, 40], device=gpu)
    lens = torch.tensor([5, 36, 20, 0, -3], device=gpu)
    cache.write(k.to(gpu), v.to(gpu), starts, table, lens)
    want = Blocks8(6, H, d)
    want.write(k[2:7], 0, 0)
    want.q[2, :10] = e4m3(torch.tensor([17], dtype=torch.uint8).view(F8).double())
    want.e[2] = 17 - 127
    want.write(k[7:13], 2, 10)
    want.write(k[33:37], 3, 0)
    slots = {0: range(0, 5), 2: range(0, 16), 3: range(0, 4)}
    raw, scales = cache.key_cache.cpu(), cache.key_scales.cpu()
    for b in range(6):
        for s in range(PAGE):
            if s in slots.get(b, ()):
                assert torch.equal(raw[b, s].double(), want.q[b, s]), (b, s)
            else:
                assert (raw[b, s].view(torch.uint8) == 17).all(), (b, s)
        assert (scales[b].double() - 127 == (want.e[b] if b in slots else 17 - 127)).all(), b
    out = cache.read(starts, table, lens, rows=60, dtype=torch.float32)[0].cpu()
    for rows in (range(0, 2), range(13, 17), range(17, 33), range(37, 60)):
        assert (out[list(rows)] == 0).all()
    assert torch.equal(out[2:7].double(), want.values()[0, :5]) and torch.equal(out[33:37].double(), want.values()[3, :4])
    given = torch.full((60, H, d), 3.0, device=gpu), torch.full((60, H, d), 4.0, device=gpu)
    assert cache.read(starts, table, lens, out=given)[0] is given[0]
    assert (given[0][40:] == 3).all() and (given[1][40:] == 4).all() and torch.equal(given[0][:40].cpu(), out[:40])


def test_many_sequences_and_one_table(gpu):
    """More sequences than a round of the search takes; most without rows."""
    B = 700
    w = Writer(gpu, [2] * B, 1, 64)
    g = torch.Generator().manual_seed(5)
    runs = torch.randint(0, 20, (B,), generator=g) * (torch.rand(B, generator=g) < 0.3)
    runs[-1] = 19
    k, v = (torch.randn(int(runs.sum()), 1, 64, generator=g).half() for _ in range(2))
    w.step(runs.tolist(), k, v)
    w.check(torch.float16)
    one = w.table[B - 1].to(gpu)
    lens, starts = torch.tensor([19], device=gpu), torch.tensor([0, 19], device=gpu)
    a = w.cache.read(starts, one, lens, rows=19)
    w.cache.write(k[-19:].to(gpu), v[-19:].to(gpu), starts, one, lens)
    assert all(torch.equal(x, y) for x, y in zip(a, w.cache.read(starts, one, lens, rows=19)))


def test_a_captured_step_is_replayed(gpu):
    """The lengths grow on the GPU; every replay writes the next token, the program's own work in between."""
    w = Writer(gpu, [3, 3], 2, 128)
    g = torch.Generator().manual_seed(6)
    w.step([10, 20], *(torch.randn(30, 2, 128, generator=g).bfloat16() for _ in range(2)))
    k, v = (torch.zeros(2, 2, 128, dtype=torch.bfloat16, device=gpu) for _ in range(2))
    lens, starts, table = torch.tensor([10, 20], dtype=torch.int32, device=gpu), torch.tensor([0, 1, 2], dtype=torch.int32, device=gpu), w.table.to(gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lens.add_(1)
        w.cache.write(k, v, starts, table, lens)
        back = w.cache.read(starts, table, lens, rows=2)
    for i in range(9):
        new = [(3.0 ** i * torch.randn(2, 2, 128, generator=g)).bfloat16() for _ in range(2)]
        k.copy_(new[0]); v.copy_(new[1])
        graph.replay()
        torch.cuda.synchronize()
        for x, want in zip(new, w.want):
            for b in range(2):
                n = w.len[b]
                want.write(x[b: b + 1], int(w.table[b, n // PAGE]), n % PAGE)
        w.len = [n + 1 for n in w.len]
        got = w.check(torch.bfloat16)
        at = torch.tensor([0] + w.len).cumsum(0)[1:] - 1
        assert torch.equal(back[0], got[0][at.to(gpu)]) and torch.equal(back[1], got[1][at.to(gpu)])


def test_another_stream_and_inference_tensors(gpu):
    w = Writer(gpu, [2], 1, 64)
    k, v = (torch.randn(20, 1, 64, generator=torch.Generator().manual_seed(7)) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.inference_mode():
        w.step([20], k, v)
        w.check()
    torch.cuda.current_stream().wait_stream(side)
    version = w.cache.key_cache._version
    w.cache.write(k.to(gpu), v.to(gpu), torch.tensor([0, 20], device=gpu), w.table.to(gpu), torch.tensor([20], device=gpu))
    assert w.cache.key_cache._version > version and w.cache.value_scales._version > 0
    w.check()


def test_blocks_of_other_layouts(gpu):
    for layout in ("engine", "heads", "padded"):
        s = Step([40, 3], [40, 3], 2, 128, "fp8", torch.bfloat16, layout=layout)
        k, v = s.cache().read(s.starts, s.table, s.seq_lens, rows=43, dtype=torch.float32)
        for b, at in ((0, slice(0, 40)), (1, slice(40, 43))):
            k64, v64, _ = s.tokens(b, s.lens[b])
            assert torch.equal(k[at].cpu().double(), k64) and torch.equal(v[at].cpu().double(), v64)
        cache = s.cache()
        cache.write(k, v, s.starts, s.table, s.seq_lens)               # what is held goes in again as it is
        again = cache.read(s.starts, s.table, s.seq_lens, rows=43, dtype=torch.float32)
        assert torch.equal(again[0], k) and torch.equal(again[1], v)
    assert LOWEST == -117
