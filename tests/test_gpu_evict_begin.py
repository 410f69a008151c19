"""Rows of tracked weights whose sequence begins in a step."""

import pytest
import torch

from turboquant_amd.eviction import begin_rows

pytestmark = pytest.mark.gpu


def held(gpu, B, H, L, strided):
    w, p = torch.rand(B, H, L, device=gpu) + 1, torch.randint(0, 99, (B, H, L), dtype=torch.int32, device=gpu)
    if strided:                                               # heads first, rows further apart than they are long
        w = torch.cat([w, w], -1).transpose(0, 1).contiguous().transpose(0, 1)[..., 1:L + 1]
        p = torch.cat([p, p], -1).transpose(0, 1).contiguous().transpose(0, 1)[..., 1:L + 1]
    return w, p


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("H,L", [(1, 1), (3, 40), (2, 4096), (2, 4097), (1, 20000)])
def test_rows_that_begin_and_the_others(gpu, H, L, strided):
    # begins with several tokens / goes on / begins with one / has no rows / is empty / a chunk that is not the first / a padded row
    lens, runs = [7, 9, 1, 0, 5, 12, 0], [7, 1, 1, 0, 0, 11, 1]
    starts = torch.tensor([3] + runs).cumsum(0)               # (rows in front of the first sequence's)
    w, p = held(gpu, 7, H, L, strided)
    w0, p0, version = w.clone(), p.clone(), w._version
    for lens_d, starts_d in ((torch.tensor(lens, dtype=torch.int32, device=gpu), starts.to(device=gpu, dtype=torch.int32)), (torch.tensor(lens), starts)):
        begin_rows(w, p, lens_d, starts_d)
        for b in range(7):
            if b in (0, 2):
                assert not w[b].any() and torch.equal(p[b].cpu(), torch.arange(L, dtype=torch.int32).expand(H, L))
            else:
                assert torch.equal(w[b], w0[b]) and torch.equal(p[b], p0[b])
    assert w._version > version


def test_refusals(gpu):
    w, p = held(gpu, 2, 2, 40, False)
    lens, starts = torch.tensor([3, 4], device=gpu), torch.tensor([0, 3, 7], device=gpu)
    begin_rows(w[:0], p[:0], lens[:0], starts[:1])
    for bad, error in ((dict(weights=w.cpu()), RuntimeError), (dict(positions=p.cpu()), RuntimeError), (dict(weights=w.double()), TypeError),
                       (dict(positions=p.long()), TypeError), (dict(weights=w[0]), ValueError), (dict(positions=p[..., :39]), ValueError),
                       (dict(weights=w[..., :20], positions=p[..., ::2]), ValueError), (dict(weights=w[:1].expand(2, 2, 40)), ValueError),
                       (dict(weights=torch._neg_view(w)), ValueError), (dict(weights=w.clone().requires_grad_()), RuntimeError),
                       (dict(seq_lens=lens[:1]), ValueError), (dict(query_start_loc=starts[:2]), ValueError)):
        with pytest.raises(error):
            begin_rows(**{**dict(weights=w, positions=p, seq_lens=lens, query_start_loc=starts), **bad})
