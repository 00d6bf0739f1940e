"""Rows of the adapters' groups that name no token, and values that are not
finite, in both forms of the kernels."""
import pytest
import torch

from oracle import adapters

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _ops():
    from zmoe import ops
    return ops


def _pad(t):
    """One more token, all zeros: what a row of no token stands for."""
    return torch.cat([t, torch.zeros(1, t.shape[1], dtype=t.dtype)])


@pytest.mark.parametrize("T,R", [(9, 16), (300, 40), (1300, 16), (1300, 104)])
def test_rows_of_no_token(T, R):
    ops = _ops()
    g = torch.Generator().manual_seed(T + R)
    G, H, N = 3, 264, 136
    tor = torch.randperm(T, generator=g).to(torch.int32)
    offsets = torch.tensor([0, T // 3, T // 2, T - 2], dtype=torch.int32)
    hole = torch.zeros(T, dtype=torch.bool)
    hole[torch.randperm(T - 2, generator=g)[:max(2, T // 10)]] = True
    hole[0] = True
    listed = torch.where(hole, torch.tensor([-1, T, 2 ** 30])[torch.arange(T) % 3], tor).to(torch.int32)
    mk = lambda *s: torch.randn(*s, generator=g).to(BF)  # noqa: E731
    x, base, dy, dx0, a, b = mk(T, H), mk(T, N), mk(T, N), mk(T, H), mk(G, R, H), mk(G, N, R)
    # the first token must not leak into rows that name none
    x[0], dy[0] = float("nan"), float("nan")
    padded = torch.where(hole, T, tor).to(torch.int32)
    kept = torch.zeros(T, dtype=torch.bool)
    kept[tor[~hole].long()] = True
    kept[0] = False

    u = torch.full((T, R), -3.0).cuda()
    cu = [t.cuda() for t in (x, base, a, b, offsets, listed)]
    out = ops.lora(cu[0], cu[1], cu[2], cu[3], None, cu[4], cu[5], out=cu[1].clone(), u=u)
    (want, bound), (uw, ub) = adapters.lora(_pad(x), _pad(base), a, b, None, offsets, padded)
    assert adapters.outside(out[kept.cuda()], want[:T][kept], bound[:T][kept])[0] == 0
    n = int(offsets[-1])
    assert (u[:n][hole[:n].cuda()] == 0).all() and (u[n:] == -3).all()
    rows = torch.tensor([r for r in range(n) if not hole[r] and tor[r] != 0])
    assert adapters.outside(u[rows.cuda()], uw[rows], ub[rows])[0] == 0

    if (listed[:n] == 0).any():                         # a NaN token of its own group: leave it out of dA and dB
        x[0], dy[0] = 0, 0
        u[(listed[:n] == 0).nonzero()[0].cuda()] = 0
    dx, da, db = ops.lora_grad(dy.cuda(), x.cuda(), u, cu[2], cu[3], None, cu[4], cu[5], base=dx0.cuda(), dx=dx0.cuda())
    ref = adapters.lora_grad(_pad(dy), _pad(x), _pad(u.cpu())[:T + 1], a, b, None, offsets, padded, base=_pad(dx0))
    assert adapters.outside(dx[kept.cuda()], ref["dx"][0][:T][kept], ref["dx"][1][:T][kept])[0] == 0
    for got, name in ((da, "da"), (db, "db")):
        assert adapters.outside(got, *ref[name])[0] == 0, name


@pytest.mark.parametrize("T,R", [(9, 16), (1300, 64), (1300, 104)])
def test_infinities_stay_where_they_belong(T, R):
    """An infinite weight or input reaches the outputs that depend on it (as an
    infinity or a NaN) and no other."""
    ops = _ops()
    g = torch.Generator().manual_seed(T * R)
    G, H, N = 2, 136, 200
    offsets, tor = torch.tensor([0, T // 2, T], dtype=torch.int32), torch.arange(T - 1, -1, -1, dtype=torch.int32)
    mk = lambda *s: torch.randn(*s, generator=g).to(BF)  # noqa: E731
    x, base, dy, a, b = mk(T, H), mk(T, N), mk(T, N), mk(G, R, H), mk(G, N, R)
    x[T - 1, 5] = float("inf")                          # in group 0
    b[1, 7, 3] = float("-inf")
    a[1, 2, 9] = float("inf")
    cu = [t.cuda() for t in (x, base, dy, a, b, offsets, tor)]
    u = torch.zeros(T, R).cuda()
    out = ops.lora(cu[0], cu[1], cu[3], cu[4], None, cu[5], cu[6], u=u).float().cpu()
    in1 = torch.zeros(T, dtype=torch.bool)
    in1[tor[T // 2:].long()] = True
    bad = torch.zeros(T, N, dtype=torch.bool)
    bad[in1], bad[T - 1] = True, True                   # a's rank reaches every column of its group's rows
    assert out.isfinite()[~bad].all() and not out.isfinite()[T - 1].any() and not out.isfinite()[in1].any()
    a[1, 2, 9] = 0
    out = ops.lora(cu[0], cu[1], a.cuda(), cu[4], None, cu[5], cu[6], u=u).float().cpu()
    bad[in1] = False
    bad[in1, 7] = True
    assert out.isfinite()[~bad].all() and not out.isfinite()[bad].any()
    dx, da, db = ops.lora_grad(cu[2], cu[0], torch.ones(T, R).cuda(), a.cuda(), cu[4], None, cu[5], cu[6])
    assert not dx.isfinite()[in1.cuda()].all(1).any() and dx.isfinite()[~in1.cuda()].all()
    ok = torch.ones(G, R, H, dtype=torch.bool)
    ok[0, :, 5], ok[1, 3] = False, False
    assert da.cpu().isfinite()[ok].all() and not da.cpu().isfinite()[~ok].any()
    assert db.isfinite().all()
