"""The token sort on both sides of the sizes at which its launches change
(1024 pairs with rows to copy, 131072 pairs), and the ways in which its one-launch
form shares the copy: all slots of a token in one CTA, some of them, or one each;
more than one piece a thread; 32 slots."""
import numpy as np
import pytest
import torch

from test_sort_grad_gpu import _idx, _plain_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,k,E,H", [(256, 4, 60, 2048), (257, 4, 60, 2048), (128, 8, 60, 2048), (1024, 1, 64, 2048),
                                     (1025, 1, 64, 2048), (32, 32, 40, 2048), (33, 32, 40, 2048), (170, 6, 64, 1032),
                                     (171, 6, 64, 1032), (3, 7, 60, 2048), (21843, 6, 64, 16), (21846, 6, 64, 16)])
@pytest.mark.parametrize("bad", [False, True])
def test_forms(T, k, E, H, bad):
    from zmoe import ops
    idx = _idx(T, k, E, 3 * T + k, bad)
    offs, tor, row_of = _plain_rows(idx, E)
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16)
    counts, offsets, r_of, t_of, xp = ops.permute(torch.from_numpy(idx).cuda(), x.cuda(), E)
    n = int(offs[-1])
    assert np.array_equal(counts.cpu().numpy(), np.diff(offs)) and np.array_equal(offsets.cpu().numpy(), offs)
    assert np.array_equal(r_of.cpu().numpy(), row_of) and np.array_equal(t_of[:n].cpu().numpy(), tor)
    assert torch.equal(xp[:n].cpu(), x[torch.from_numpy(tor).long()])
