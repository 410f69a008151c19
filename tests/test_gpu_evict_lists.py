"""tq_evict_select as C callers reach it: lists of moves longer than there can be moves, in rows of one workgroup and of several."""

import pytest
import torch

from tests.exact_helpers import evict64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("L,budget", [(300, 100), (9000, 4000), (20000, 300), (17000, 16990)])
@pytest.mark.parametrize("more", [0, 1, 1500, 30000])
def test_lists_end_in_minus_one(gpu, L, budget, more):
    from turboquant_amd import _ffi
    B, H, least = 3, 2, max(1, min(budget, L - budget))
    moves = least + more
    g = torch.Generator().manual_seed(L + more)
    w, pos = torch.rand(B, H, L, generator=g), torch.arange(L, dtype=torch.int32).expand(B, H, L).contiguous()
    held = [L, budget, 0]
    want = evict64(w, pos, held, None, budget, 4, 16)
    whole = lambda *shape: torch.full(shape, 77, dtype=torch.int32, device=gpu)
    lens, count, dst, src, new_p = whole(B), whole(B, H), whole(B, H, moves), whole(B, H, moves), whole(B, H, L)
    new_w, w_d, p_d, l_d = torch.empty(B, H, L, device=gpu), w.to(gpu), pos.to(gpu), torch.tensor(held, dtype=torch.int32, device=gpu)
    lib = _ffi.lib()
    need = lib.tq_evict_select_bytes(B, H, L, budget, moves)
    workspace = torch.empty(max(1, need // 4), device=gpu)
    assert lib.tq_evict_select(w_d.data_ptr(), H * L, L, p_d.data_ptr(), H * L, L, l_d.data_ptr(), None, B, H, L, budget, 4, 16, moves, lens.data_ptr(),
                               count.data_ptr(), dst.data_ptr(), src.data_ptr(), new_w.data_ptr(), H * L, L, new_p.data_ptr(), H * L, L,
                               workspace.data_ptr(), _ffi.stream_ptr(gpu)) == 0
    for got, x in zip((lens, count, dst[..., :least], src[..., :least], new_w, new_p), want):
        assert torch.equal(got.cpu(), x)
    assert (dst[..., least:] == -1).all() and (src[..., least:] == -1).all()
