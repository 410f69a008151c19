"""Sizes that the eviction's entry points refuse before they launch anything: no GPU is touched."""

from tests.test_exact_host import select_args
from turboquant_amd import _ffi


def test_lists_of_moves_that_an_index_could_not_count():
    for L in (40, 40000):
        for moves in (2 ** 30 + 1, 2 ** 31 - 1):
            assert _ffi.lib().tq_evict_select(*select_args(L=L, moves=moves, workspace=1 << 20)) == -1


def test_rows_that_begin():
    P = 1 << 20
    ok = dict(w=P, w_b=80, w_h=40, pos=P, p_b=80, p_h=40, lens=P, starts=P, B=0, H=2, L=40, stream=None)
    call = lambda **kw: _ffi.lib().tq_evict_begin(*{**ok, **kw}.values())
    assert call() == 0
    for bad, rc in ((dict(w=None), -3), (dict(pos=None), -3), (dict(lens=None), -3), (dict(starts=None), -3), (dict(B=-1), -1), (dict(H=0), -1), (dict(L=0), -1),
                    (dict(L=2 ** 30 + 1), -1), (dict(w_b=-1), -1), (dict(p_h=-1), -1), (dict(B=2 ** 20, H=2 ** 11), -1), (dict(B=2 ** 20, L=2 ** 30), -1)):
        assert call(**bad) == rc, bad
