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


@pytest.mark.parametrize("T,k", [(1, 4), (5, 3), (900, 6)])
@pytest.mark.parametrize("capacity", [0, 1])
def test_same_without_the_compiled_module(T, k, capacity, monkeypatch):
    ops = _ops()
    g = torch.Generator().manual_seed(T)
    k = 1 if capacity else k
    idx = torch.stack([torch.randperm(9, generator=g)[:k] for _ in range(T)]).to(torch.int32).cuda()
    x = torch.randn(T, 72, generator=g).to(torch.bfloat16).cuda()
    for xd in (x, None):
        i, j = idx.clone(), idx.clone()
        want = ops.permute(i, xd, 9, capacity, T)
        with monkeypatch.context() as m:
            m.setattr(ops, "_ops", None)
            got = ops.permute(j, xd, 9, capacity, T)
        assert torch.equal(i, j) and (want[4] is None) == (got[4] is None)
        n = int(want[1][-1])
        for p, q in zip(want[:3], got[:3]):
            assert torch.equal(p, q)
        assert torch.equal(want[3][:n], got[3][:n])
        if xd is not None:
            assert torch.equal(want[4][:n], got[4][:n])
