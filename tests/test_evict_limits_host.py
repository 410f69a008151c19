"""Sizes that the eviction's entry points refuse before they launch anything: no GPU is touched."""

from tests.test_exact_host import select_args
from turboquant_amd import _ffi


def test_lists_of_moves_that_an_index_could_not_count():
    for L in (40, 40000):
        for moves in (2 ** 30 + 1, 2 ** 31 - 1):
            assert _ffi.lib().tq_evict_select(*select_args(L=L, moves=moves, workspace=1 << 20)) == -1
