"""What the Python calls of a step hand to the library and what they refuse before, on host tensors: the library is a list of the calls it gets."""

import contextlib

import pytest
import torch

from turboquant_amd import _ffi
from turboquant_amd.rotary import inverse_frequencies, rotate_heads


@pytest.fixture
def calls(monkeypatch):
    got, real = [], _ffi.lib()

    class Library:
        def __getattr__(self, name):
            return getattr(real, name) if name.endswith("_bytes") else lambda *a: got.append((name, a)) or 0
    monkeypatch.setattr(_ffi, "lib", Library)
    monkeypatch.setattr(_ffi, "native", lambda: None)
    monkeypatch.setattr(_ffi, "require_gpu", lambda t, name: t)
    monkeypatch.setattr(_ffi, "on_device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(_ffi, "stream_ptr", lambda device: None)
    return got


# ---- rotation in place ------------------------------------------------------------------------------------------------------------

def heads(rows=6, H=4, d=64):
    """Queries and keys of as many heads, and the two as views of one projection."""
    q, k = torch.zeros(rows, H, d), torch.zeros(rows, H, d)
    qkv = torch.zeros(rows, 3 * H * d)
    return (q, k), (qkv[:, : H * d].view(rows, H, d), qkv[:, H * d: 2 * H * d].view(rows, H, d))


def rotate(q, k, out):
    return rotate_heads(q, k, torch.arange(q.shape[0]), inverse_frequencies(q.shape[2]), out=out)


@pytest.mark.parametrize("views", [False, True])
def test_an_output_replaces_its_own_input_only(calls, views):
    """A head is read by the lanes that write it, and by nobody before: true of out=(query, key), not of an output in the other input's place."""
    q, k = heads()[views]
    for out in ((k, q), (k, torch.zeros_like(q)), (torch.zeros_like(q), q), (k, k.clone()), (q.clone(), q)):
        with pytest.raises(ValueError):
            rotate(q, k, out)
    assert not calls
    allowed = (q, k), (q, torch.zeros_like(k)), (torch.zeros_like(q), k)
    for out in allowed:
        assert rotate(q, k, out)[0] is out[0]
    assert [(a[0], a[1], a[19], a[22]) for _, a in calls] == [tuple(t.data_ptr() for t in (q, k, *out)) for out in allowed]


def test_queries_that_are_the_keys(calls):
    """One tensor, or two that share heads: neither may be written."""
    q, new = heads()[0]
    wide = torch.zeros(6, 6, 64)
    for a, b in ((q, q), (wide[:, :4], wide[:, 2:])):
        for out in ((a, new), (new, b), (a, b)):
            with pytest.raises(ValueError):
                rotate(a, b, out)
        assert not calls
        rotate(a, b, (new, new.clone()))
        rotate(a, b, None)
        assert len(calls) == 2
        calls.clear()


def test_outputs_beside_inputs_of_one_projection(calls):
    """Columns that nobody reads may be written."""
    rows, H, d = 6, 4, 64
    x = torch.zeros(rows, 4 * H * d)
    q, k, a, b = (x[:, i * H * d: (i + 1) * H * d].view(rows, H, d) for i in range(4))
    for out in ((a, b), (q, a), (a, k), (q, k)):
        rotate(q, k, out)
    assert len(calls) == 4
    for out in ((a, a), (k, a), (a, q), (x[:, 64: 64 + H * d].view(rows, H, d), k)):
        with pytest.raises(ValueError):
            rotate(q, k, out)
    assert len(calls) == 4
