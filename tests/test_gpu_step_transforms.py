"""Calls of a step's operators that torch is differentiating, transforming or recording: refused, since the result would be a constant; and under modes that only
watch, the same as without."""

import pytest
import torch
import torch.autograd.forward_ad as fwad
from torch.overrides import TorchFunctionMode
from torch.utils._python_dispatch import TorchDispatchMode

from tests.step_helpers import Step
from turboquant_amd.fp8 import Fp8PagedCache
from turboquant_amd.rotary import inverse_frequencies, rotate_heads

pytestmark = pytest.mark.gpu


class Case:
    """One object for each call: its tensors by name, the calls, and what they may write."""

    def __init__(self, gpu, kind):
        self.step = Step([70, 40], [3, 1], 2, 64, "fp8" if kind == "fp8" else torch.bfloat16, torch.bfloat16)
        self.kc, self.vc = (x.view(torch.uint8).clone().view(x.dtype) if kind == "fp8" else x.nan_to_num() for x in self.step.q)
        g = torch.Generator().manual_seed(1)
        self.q = self.step.query(4).to(gpu)
        self.k, self.v = (torch.randn(4, 2, 64, generator=g).bfloat16().to(gpu) for _ in range(2))
        self.w, self.f, self.pos = torch.rand(64, generator=g).bfloat16().to(gpu), inverse_frequencies(64, device=gpu), torch.arange(4, device=gpu)
        self.out_q, self.out_k = torch.zeros_like(self.q), torch.zeros_like(self.k)
        self.kind = kind

    def cache(self, a):
        if self.kind == "fp8":
            return Fp8PagedCache(a["kc"], a["vc"], *self.step.scales)
        from turboquant_amd.exact import ExactPagedCache
        return ExactPagedCache(a["kc"], a["vc"])

    def attention(self, **kw):
        a, s = {**vars(self), **kw}, self.step
        return self.cache(a).attention(a["q"], s.starts, s.table, s.seq_lens, window=30)

    def attention_out(self, **kw):
        a, s = {**vars(self), **kw}, self.step
        return self.cache(a).attention(a["q"], s.starts, s.table, s.seq_lens, window=30, out=a["out_q"])

    def decode(self, **kw):
        a, s = {**vars(self), **kw}, self.step
        return self.cache(a).decode_attention(a["q"][:2], s.table, s.seq_lens, window=30)

    def write(self, **kw):
        a, s = {**vars(self), **kw}, self.step
        self.cache(a).write(a["k"], a["v"], s.starts, s.table, s.seq_lens)
        return a["kc"].view(torch.uint8).clone()

    def read(self, **kw):
        a, s = {**vars(self), **kw}, self.step
        return self.cache(a).read(s.starts, s.table, s.seq_lens, rows=4)

    def read_out(self, **kw):
        a, s = {**vars(self), **kw}, self.step
        return self.cache(a).read(s.starts, s.table, s.seq_lens, out=(a["out_k"], a["v"]))

    def rotate(self, **kw):
        a = {**vars(self), **kw}
        return rotate_heads(a["q"], a["k"], self.pos, a["f"], a["w"], a["w"])

    def rotate_out(self, **kw):
        a = {**vars(self), **kw}
        return rotate_heads(a["q"], a["k"], self.pos, a["f"], a["w"], a["w"], out=(a["out_q"], a["out_k"]))

    def held(self):
        return [t.view(torch.uint8).clone() for t in (self.kc, self.vc, self.q, self.k, self.v, self.out_q, self.out_k, *(self.step.scales if self.kind == "fp8" else ()))]


PARTS = [("bf16", n, p) for n in ("attention", "decode") for p in ("q", "kc", "vc")] + [("bf16", "attention_out", "out_q"), ("fp8", "attention", "q"), ("fp8", "decode", "q"),
         ("fp8", "write", "k"), ("fp8", "write", "v"), ("fp8", "read_out", "out_k"), ("fp8", "rotate", "q"), ("fp8", "rotate", "k"), ("fp8", "rotate", "w"), ("fp8", "rotate", "f"),
         ("fp8", "rotate_out", "out_q"), ("fp8", "rotate_out", "out_k")]
CALLS = [("bf16", "attention"), ("bf16", "decode"), ("fp8", "attention"), ("fp8", "decode"), ("fp8", "write"), ("fp8", "read"), ("fp8", "rotate")]


def refused(c, call):
    before = c.held()
    with pytest.raises(RuntimeError):
        call()
    assert all(torch.equal(a, b) for a, b in zip(before, c.held()))


@pytest.mark.parametrize("kind,name,part", PARTS)
def test_a_tangent(gpu, kind, name, part):
    c = Case(gpu, kind)
    with fwad.dual_level():
        t = getattr(c, part)
        dual = fwad.make_dual(t.clone(), torch.ones_like(t))
        refused(c, lambda: getattr(c, name)(**{part: dual}))
        getattr(c, name)()                                    # (none among the arguments)


@pytest.mark.parametrize("kind,name,part", PARTS)
def test_a_gradient(gpu, kind, name, part):
    c = Case(gpu, kind)
    t = getattr(c, part).clone().requires_grad_()
    refused(c, lambda: getattr(c, name)(**{part: t}))
    with torch.no_grad():
        getattr(c, name)(**{part: t})


@pytest.mark.parametrize("kind,name", CALLS)
def test_a_trace(gpu, kind, name):
    c = Case(gpu, kind)

    def traced(x):
        getattr(c, name)()
        return x + 1
    refused(c, lambda: torch.jit.trace(traced, (c.w,), check_trace=False))


@pytest.mark.parametrize("kind,name,part", [p for p in PARTS if p[2] in "qkw"])
def test_a_batch_of_calls(gpu, kind, name, part):
    """vmap's tensors have no memory of their own."""
    c = Case(gpu, kind)
    t = getattr(c, part)
    refused(c, lambda: torch.vmap(lambda x: getattr(c, name)(**{part: x}))(torch.stack([t, t])))


class Dispatch(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


class Function(TorchFunctionMode):
    def __torch_function__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("kind,name", CALLS)
@pytest.mark.parametrize("mode", [Dispatch, Function, torch.inference_mode, torch.no_grad])
def test_modes_that_watch(gpu, kind, name, mode):
    bits = lambda x: [t.view(torch.uint8) for t in (x if isinstance(x, tuple) else (x,))]
    want = bits(getattr(Case(gpu, kind), name)())
    c = Case(gpu, kind)
    with mode():
        got = getattr(c, name)()
    assert all(torch.equal(a, b) for a, b in zip(want, bits(got)))


@pytest.mark.parametrize("kind,name", CALLS)
def test_new_memory_that_is_filled(gpu, kind, name):
    want = getattr(Case(gpu, kind), name)()
    torch.use_deterministic_algorithms(True)
    try:
        got = getattr(Case(gpu, kind), name)()
    finally:
        torch.use_deterministic_algorithms(False)
    assert all(torch.equal(a, b) for a, b in zip(want if isinstance(want, tuple) else (want,), got if isinstance(got, tuple) else (got,)))
