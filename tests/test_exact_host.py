"""What the exact cache's entry points refuse before they launch anything, and their plans: no GPU is touched."""

import ctypes as C

import pytest
import torch

from turboquant_amd import _ffi

P = 1 << 20                                  # an aligned address that no refused call looks at


def decode_args(**kw):
    a = dict(q=P, dtype=2, B=2, Hq=8, Hkv=2, d=128, k=P, v=P, cs_blk=16 * 256, cs_t=256, cs_h=128, num_blocks=4, table=P, bt_stride=2, lens=P,
             scale=0.1, max_len=32, weights=None, w_b=64, w_h=32, weight_len=32, out=P, workspace=P, n_split=0, stream=None)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


@pytest.mark.parametrize("bad,rc", [
    (dict(q=None), -3), (dict(out=None), -3), (dict(k=None), -3), (dict(v=None), -3), (dict(table=None), -3), (dict(lens=None), -3),
    (dict(workspace=None), -3), (dict(dtype=3), -1), (dict(dtype=-1), -1), (dict(B=-1), -1), (dict(Hq=0), -1), (dict(Hkv=0), -1),
    (dict(Hq=9), -1), (dict(d=96), -1), (dict(d=0), -1), (dict(d=832), -1), (dict(num_blocks=0), -1), (dict(bt_stride=0), -1),
    (dict(bt_stride=-2 ** 31), -1), (dict(max_len=-1), -1), (dict(n_split=-1), -1), (dict(n_split=1025), -1),
    (dict(Hq=2 * 1025, n_split=1), -1), (dict(weights=P, w_b=-1), -1), (dict(weights=P, weight_len=-1), -1),
    (dict(cs_t=-256), -2), (dict(cs_t=(1 << 24) + 8), -2), (dict(cs_t=257), -2), (dict(cs_blk=4097), -2), (dict(cs_h=4), -2),
    (dict(k=P + 2), -2), (dict(v=P + 8), -2), (dict(q=P + 2), -2), (dict(out=P + 4), -2), (dict(workspace=P + 4), -1),
])
def test_decode_refuses(bad, rc):
    assert _ffi.lib().tq_exact_decode(*decode_args(**bad)) == rc


def test_decode_of_nothing_launches_nothing():
    assert _ffi.lib().tq_exact_decode(*decode_args(B=0, workspace=None)) == 0


def test_decode_plans():
    need = _ffi.lib().tq_exact_decode_bytes
    assert need(2, 2, 8, 2, 96, 32, 0, 0) == 0 and need(2, 2, 9, 2, 128, 32, 0, 0) == 0 and need(2, 2, 8, 2, 128, -1, 0, 0) == 0
    base = need(2, 2, 8, 2, 128, 4096, 1, 0)
    assert base > 0
    # a split more: its numerators, maximum and sum
    assert need(2, 2, 8, 2, 128, 4096, 4, 0) - need(2, 2, 8, 2, 128, 4096, 2, 0) == 2 * 16 * (128 * 4 + 8)
    # scores of every head and token, for the weights
    assert need(2, 2, 8, 2, 128, 4096, 1, 4096) - base == 2 * 8 * 4096 * 4
    # more workgroups than a grid holds
    assert need(2, 2 ** 20, 1024, 1024, 128, 1 << 22, 1024, 0) == 0


def test_a_cache_on_the_host_is_refused():
    from turboquant_amd.exact import ExactPagedCache
    t = torch.zeros(2, 4, 16, 2, 64)
    with pytest.raises(RuntimeError):
        ExactPagedCache.from_engine(t)
