"""Calls of the exact cache's operators that torch is differentiating or recording: refused, since the result would be a constant of either."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

from tests.exact_helpers import Sequences
from turboquant_amd.eviction import begin_rows, select_evictions
from turboquant_amd.exact import ExactPagedCache

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, gpu):
        self.seqs = Sequences([70, 40], 2, 64, torch.float32)
        self.seqs.kv.nan_to_num_()
        self.k, self.v = self.seqs.kv[0].clone(), self.seqs.kv[1].clone()
        self.q, self.w = self.seqs.query(2, 4, 64).to(gpu), torch.rand(2, 2, 80, device=gpu)
        self.pos = torch.arange(80, dtype=torch.int32, device=gpu).expand(2, 2, 80).contiguous()
        self.starts = torch.tensor([0, 1, 2], dtype=torch.int32, device=gpu)
        self.cut = select_evictions(self.w, self.pos, self.seqs.seq_lens, 20)

    def decode(self, **kw):
        a = {**vars(self), **kw}
        return ExactPagedCache(a["k"], a["v"]).decode_attention(a["q"], self.seqs.table, self.seqs.seq_lens, weights=a["w"])

    def window(self, **kw):
        a = {**vars(self), **kw}
        return ExactPagedCache(a["k"], a["v"]).add_window_weights(a["q"], self.starts, self.seqs.table, self.seqs.seq_lens, a["w"], 4)

    def select(self, **kw):
        return select_evictions({**vars(self), **kw}["w"], self.pos, self.seqs.seq_lens, 20)

    def begin(self, **kw):
        begin_rows({**vars(self), **kw}["w"], self.pos, self.seqs.seq_lens, self.starts)

    def move(self, **kw):
        a = {**vars(self), **kw}
        ExactPagedCache(a["k"], a["v"]).move_tokens(self.cut, self.seqs.table)


PARTS = [("decode", "q"), ("decode", "k"), ("decode", "v"), ("decode", "w"), ("window", "q"), ("window", "k"), ("window", "w"), ("begin", "w"),
         ("move", "k"), ("move", "v")]


def unchanged(c, call):
    held = [t.clone() for t in (c.k, c.v, c.w, c.pos)]
    with pytest.raises(RuntimeError):
        call()
    assert all(torch.equal(a, b) for a, b in zip(held, (c.k, c.v, c.w, c.pos)))


@pytest.mark.parametrize("name,part", PARTS)
def test_a_tangent(gpu, name, part):
    c = Case(gpu)
    getattr(c, name)()
    with fwad.dual_level():
        t = getattr(c, part)
        dual = fwad.make_dual(t, torch.ones_like(t))
        unchanged(c, lambda: getattr(c, name)(**{part: dual}))
        getattr(c, name)()                                    # (none among the arguments)
    getattr(c, name)()


@pytest.mark.parametrize("name,part", PARTS)
def test_a_gradient(gpu, name, part):
    c = Case(gpu)
    t = getattr(c, part).clone().requires_grad_()
    unchanged(c, lambda: getattr(c, name)(**{part: t}))
    with torch.no_grad():
        getattr(c, name)(**{part: t})


def test_select_takes_weights_as_numbers(gpu):
    """Who stays is no differentiable function of the weights: the result has neither history nor tangent."""
    c = Case(gpu)
    e = c.select(w=c.w.clone().requires_grad_())
    assert not e.weights.requires_grad and torch.equal(e.weights, c.cut.weights)
    with fwad.dual_level():
        e = c.select(w=fwad.make_dual(c.w, torch.ones_like(c.w)))
        assert fwad.unpack_dual(e.weights).tangent is None and torch.equal(e.weights, c.cut.weights)


@pytest.mark.parametrize("name", ["decode", "window", "select", "begin", "move"])
def test_a_trace(gpu, name):
    c = Case(gpu)

    def traced(w):
        getattr(c, name)(w=w)
        return w + 1
    unchanged(c, lambda: torch.jit.trace(traced, (c.w,), check_trace=False))
