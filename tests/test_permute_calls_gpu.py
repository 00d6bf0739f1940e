"""Calls of ops.permute that worked before it moved to C++."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _ops():
    from zmoe import ops
    return ops


@pytest.mark.parametrize("T", [3, 700])
def test_rows_behind_the_last_token(T):
    ops = _ops()
    g = torch.Generator().manual_seed(T)
    idx = torch.stack([torch.randperm(9, generator=g)[:2] for _ in range(T)]).to(torch.int32).cuda()
    buf = torch.randn(T + 13, 72, generator=g).to(torch.bfloat16).cuda()
    want = ops.permute(idx, buf[:T].clone(), 9)
    got = ops.permute(idx, buf, 9)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    with pytest.raises(ValueError, match="row for each token"):
        ops.permute(idx, buf[:T - 1], 9)
