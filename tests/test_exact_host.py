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


def window_args(**kw):
    a = dict(q=P, dtype=2, rows=16, starts=P, B=2, Hq=8, Hkv=2, d=128, window=8, k=P, cs_blk=16 * 256, cs_t=256, cs_h=128, num_blocks=4,
             table=P, bt_stride=2, lens=P, scale=0.1, max_len=32, weights=P, w_b=64, w_h=32, weight_len=32, workspace=P, stream=None)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


@pytest.mark.parametrize("bad,rc", [
    (dict(q=None), -3), (dict(starts=None), -3), (dict(weights=None), -3), (dict(k=None), -3), (dict(lens=None), -3), (dict(workspace=None), -3),
    (dict(window=0), -1), (dict(window=1025), -1), (dict(rows=-1), -1), (dict(Hq=7), -1), (dict(d=65), -1), (dict(weight_len=0), -1),
    (dict(w_h=-1), -1), (dict(max_len=-1), -1), (dict(bt_stride=0), -1), (dict(workspace=P + 8), -1), (dict(q=P + 8), -2), (dict(k=P + 4), -2),
    (dict(cs_t=100), -2), (dict(dtype=7), -1), (dict(Hq=1 << 20, Hkv=1 << 12), -1),
])
def test_window_refuses(bad, rc):
    assert _ffi.lib().tq_exact_window(*window_args(**bad)) == rc


def test_window_of_nothing_launches_nothing():
    assert _ffi.lib().tq_exact_window(*window_args(rows=0)) == 0
    assert _ffi.lib().tq_exact_window(*window_args(B=0, workspace=None)) == 0


def select_args(**kw):
    a = dict(w=P, w_b=80, w_h=40, pos=P, p_b=80, p_h=40, lens=P, seen=None, B=2, H=2, L=40, budget=20, sinks=4, recent=3, moves=20, lens_out=P, count=P,
             dst=P, src=P, w_out=P, wo_b=80, wo_h=40, pos_out=P, po_b=80, po_h=40, workspace=None, stream=None)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


@pytest.mark.parametrize("bad,rc", [
    *((dict([(n, None)]), -3) for n in ("w", "pos", "lens", "lens_out", "count", "dst", "src", "w_out", "pos_out")),
    (dict(B=-1), -1), (dict(H=0), -1), (dict(L=0), -1), (dict(budget=0), -1), (dict(sinks=-1), -1), (dict(recent=-1), -1),
    (dict(sinks=10, recent=11), -1), (dict(sinks=2 ** 31 - 1, recent=2 ** 31 - 1), -1), (dict(moves=19), -1), (dict(w_b=-1), -1), (dict(po_h=-1), -1),
    (dict(B=2 ** 20, H=2 ** 12), -1), (dict(L=2 ** 30 + 1, budget=1, sinks=0, recent=0), -1), (dict(L=40000), -3), (dict(L=40000, workspace=P + 8), -1),
])
def test_select_refuses(bad, rc):
    assert _ffi.lib().tq_evict_select(*select_args(**bad)) == rc


def test_moves_refuse():
    exact = dict(k=P, v=P, dtype=2, d=128, cs_blk=16 * 256, cs_t=256, cs_h=128, num_blocks=4, table=P, bt_stride=2, count=P, dst=P, src=P, B=2, H=2,
                 moves=20, stream=None)
    call = lambda **kw: _ffi.lib().tq_move_tokens_exact(*{**exact, **kw}.values())
    for bad, rc in ((dict(k=None), -3), (dict(count=None), -3), (dict(dtype=4), -1), (dict(d=0), -1), (dict(bt_stride=0), -1), (dict(moves=-1), -1),
                    (dict(num_blocks=0), -1), (dict(d=100), -2), (dict(cs_t=4), -2), (dict(cs_h=-128), -2), (dict(v=P + 8), -2)):
        assert call(**bad) == rc, bad
    assert call(B=0) == 0 and call(moves=0) == 0
    layout = _ffi.make_page_layout(128, 2, 4, 32, torch.bfloat16)
    pool = dict(pool=P, num_pages=4, layout=C.byref(layout), table=P, bt_stride=2, count=P, dst=P, src=P, B=2, H=2, moves=20, budget=20, stream=None)
    call = lambda **kw: _ffi.lib().tq_move_tokens_pool(*{**pool, **kw}.values())
    for bad, rc in ((dict(pool=None), -3), (dict(layout=None), -3), (dict(table=None), -3), (dict(budget=0), -1), (dict(num_pages=0), -1)):
        assert call(**bad) == rc, bad
    assert call(B=0) == 0
