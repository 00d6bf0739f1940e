"""The token sort at the sizes where its launches change, and the gradients of
permute and combine, against plain statements (64 bits for what is computed)."""
import numpy as np
import pytest
import torch

from oracle import adapters, moe

pytestmark = pytest.mark.gpu


def _ops():
    from zmoe import ops
    return ops


def _idx(T, k, E, seed, bad=False):
    rng = np.random.default_rng(seed)
    p = 1.0 / np.arange(1, E + 1)
    u = np.log(p)[None, :] + rng.gumbel(size=(T, E))
    idx = np.argsort(-u, axis=1)[:, :k].astype(np.int32)
    if bad:                                             # no expert, and one expert twice
        idx[rng.random((T, k)) < 0.2] = -1
        idx[rng.random((T, k)) < 0.05] = E + 3
        if k > 1:
            twice = rng.random(T) < 0.2
            idx[twice, k - 1] = idx[twice, 0]
    return idx


def _plain_rows(idx, E):
    """Rows by expert, tokens ascending; an expert named twice by a token counts
    once, at its first slot."""
    T, k = idx.shape
    row_of = np.full((T, k), -1, np.int32)
    tor, offs = [], [0]
    for e in range(E):
        for t in np.nonzero((idx == e).any(1))[0]:
            row_of[t, int(np.nonzero(idx[t] == e)[0][0])] = len(tor)
            tor.append(t)
        offs.append(len(tor))
    return np.array(offs, np.int32), np.array(tor, np.int32), row_of


# T x k around 2048 pairs (one launch or two), a warp's steps, 32 slots, 1024 experts
@pytest.mark.parametrize("T,k,E,H", [(1, 1, 1, 8), (1, 4, 60, 2048), (7, 6, 64, 264), (512, 4, 60, 2048), (513, 4, 60, 256),
                                     (511, 1, 128, 1024), (5000, 6, 64, 64), (20000, 8, 60, 8), (40, 31, 33, 16),
                                     (40, 32, 40, 16), (40, 33, 40, 16), (3000, 2, 1024, 8), (300, 2, 1025, 8)])
@pytest.mark.parametrize("bad", [False, True])
def test_sort_matches_plain(T, k, E, H, bad):
    ops = _ops()
    idx = _idx(T, k, E, T + k, bad)
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16)
    offs, tor, row_of = _plain_rows(idx, E)
    if not bad:
        assert all(np.array_equal(p, q) for p, q in zip(moe.permute(idx, E), (offs, tor, row_of)))
    for xd in (x.cuda(), None):
        d = torch.from_numpy(idx).cuda()
        counts, offsets, r_of, t_of, xp = ops.permute(d, xd, E)
        assert np.array_equal(d.cpu().numpy(), idx)
        assert np.array_equal(counts.cpu().numpy(), np.diff(offs))
        assert np.array_equal(offsets.cpu().numpy(), offs)
        assert np.array_equal(r_of.cpu().numpy(), row_of)
        n = int(offs[-1])
        assert np.array_equal(t_of[:n].cpu().numpy(), tor)
        if xd is not None:
            assert torch.equal(xp[:n].cpu(), x[torch.from_numpy(tor).long()])


def test_sort_leaves_rows_behind_the_last():
    from zmoe._lib import PermuteArgs, check, lib
    import ctypes
    for T in (9, 1200):
        k, E, H = 2, 4, 64
        idx = torch.full((T, k), -1, dtype=torch.int32)
        idx[::3, 0] = 2
        n = len(range(0, T, 3))
        d, x = idx.cuda(), torch.ones(T, H, dtype=torch.bfloat16).cuda()
        counts, offsets = torch.empty(E, dtype=torch.int32).cuda(), torch.empty(E + 1, dtype=torch.int32).cuda()
        row_of = torch.empty(T, k, dtype=torch.int32).cuda()
        tor = torch.full((T * k,), -7, dtype=torch.int32).cuda()
        xp = torch.full((T * k, H), 5.0, dtype=torch.bfloat16).cuda()
        a = PermuteArgs(d.data_ptr(), x.data_ptr(), T, H, E, k, 0, 0, counts.data_ptr(), offsets.data_ptr(),
                        row_of.data_ptr(), tor.data_ptr(), xp.data_ptr())
        check(lib.zmoe_permute(ctypes.byref(a), torch.cuda.current_stream().cuda_stream), "zmoe_permute")
        assert (xp[:n] == 1).all() and (xp[n:] == 5).all() and (tor[n:] == -7).all()


def _rows(T, k, E, seed, bad=False):
    offs, tor, row_of = _plain_rows(_idx(T, k, E, seed, bad), E)
    return torch.from_numpy(row_of), int(offs[-1])


@pytest.mark.parametrize("T,k,E,H", [(1, 1, 1, 8), (3, 8, 60, 2048), (67, 6, 64, 1032), (130, 9, 20, 40), (33, 4, 8, 4096)])
@pytest.mark.parametrize("bad", [False, True])
@pytest.mark.parametrize("base", [None, "add", "in place"])
def test_permute_grad(T, k, E, H, bad, base):
    ops = _ops()
    g = torch.Generator().manual_seed(T * 31 + k)
    row_of, rows = _rows(T, k, E, T + 1, bad)
    dxp = torch.randn(rows + 2, H, generator=g).to(torch.bfloat16)
    dxp[rows:] = float("nan")                           # rows that no slot names are not read
    add = torch.randn(T, H, generator=g).to(torch.bfloat16) if base else None
    ad = add.cuda() if base else None
    dx = ops.permute_grad(dxp.cuda(), row_of.cuda(), base=ad, dx=ad if base == "in place" else None)
    want, bound = adapters.permute_grad(dxp, row_of, add)
    assert adapters.outside(dx, want, bound)[0] == 0


@pytest.mark.parametrize("mode,shared,gate", [(0, False, False), (0, True, True), (1, True, False), (2, False, False)])
@pytest.mark.parametrize("T,k,E,H", [(1, 1, 1, 8), (5, 4, 60, 2048), (67, 6, 64, 1032), (33, 3, 8, 4104)])
@pytest.mark.parametrize("bad", [False, True])
def test_combine_grad(mode, shared, gate, T, k, E, H, bad):
    ops = _ops()
    if mode == 2:
        k = 1
    g = torch.Generator().manual_seed(T * 17 + k + mode)
    row_of, rows = _rows(T, k, E, T + 2, bad)
    bf = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16)  # noqa: E731
    dout, y, w = bf(T, H), bf(rows + 3, H), torch.rand(T, k, generator=g)
    y[rows:] = float("inf")
    ysh = bf(T, H) if shared else None
    gt = torch.rand(T, generator=g) if gate else None
    x = bf(T, H) if mode == 2 else None
    dy = torch.full((rows + 3, H), 9.0, dtype=torch.bfloat16).cuda()
    cu = lambda t: None if t is None else t.cuda()  # noqa: E731
    got = ops.combine_grad(dout.cuda(), y.cuda(), row_of.cuda(), w.cuda(), mode, cu(ysh), cu(gt), cu(x), dy=dy)
    want = adapters.combine_grad(dout, y, row_of, w, mode == 2, ysh, gt, x)
    named = dict(zip(("dy", "dw", "dysh", "dg", "dx"), got))
    assert (named["dy"][rows:] == 9).all()
    assert adapters.outside(named["dy"][:rows], want["dy"][0][:rows], want["dy"][1][:rows])[0] == 0
    for n in ("dw", "dysh", "dg", "dx"):
        if named[n] is None:
            assert n not in want or (n == "dg" and not gate)
        else:
            assert adapters.outside(named[n], *want[n])[0] == 0, n


def test_combine_grad_against_differences():
    # the combine is linear in the weights, in y and in the shared rows: central
    # differences of its 64-bit statement are exact up to their own rounding
    ops = _ops()
    T, k, E, H = 6, 3, 5, 64
    g = torch.Generator().manual_seed(5)
    row_of, rows = _rows(T, k, E, 8)
    bf = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16)  # noqa: E731
    dout, y, ysh, w, gt = bf(T, H), bf(rows, H), bf(T, H), torch.rand(T, k, generator=g), torch.rand(T, generator=g)
    dy, dw, dysh, dg, _ = ops.combine_grad(dout.cuda(), y.cuda(), row_of.cuda(), w.cuda(), 0, ysh.cuda(), gt.cuda())
    loss = lambda y, w, s, q: (adapters.combine(y, row_of, w, y_shared=s, gate=q) * dout.double()).sum()  # noqa: E731
    want = adapters.combine_grad(dout, y, row_of, w, False, ysh, gt)
    args = [y.double(), w.double(), ysh.double(), gt.double()]
    for i, (got, name) in enumerate(zip((dy, dw, dysh, dg), ("dy", "dw", "dysh", "dg"))):
        d = torch.randn(args[i].shape, generator=g, dtype=torch.float64)
        hi, lo = list(args), list(args)
        hi[i], lo[i] = args[i] + d, args[i] - d
        num = (loss(*hi) - loss(*lo)) / 2
        half = torch.finfo(got.dtype).eps / 2
        tol = ((want[name][1] * 2 + half * want[name][0].abs()) * d.abs()).sum() + 1e-9
        assert abs((got.cpu().double() * d).sum() - num) <= tol, name


def test_grads_refuse():
    ops = _ops()
    d = torch.zeros(4, 16, dtype=torch.bfloat16).cuda()
    row = torch.zeros(4, 1, dtype=torch.int32).cuda()
    w = torch.ones(4, 1).cuda()
    with pytest.raises(ValueError):
        ops.permute_grad(d.float(), row)
    with pytest.raises(ValueError):
        ops.permute_grad(d, row.cpu())
    with pytest.raises(ValueError):
        ops.permute_grad(d[:, ::2], row)
    with pytest.raises(ValueError):
        ops.permute_grad(d, row, base=d[:2])
    with pytest.raises(ops._lib.ZmoeError, match="multiple of 8"):
        ops.permute_grad(torch.zeros(4, 12, dtype=torch.bfloat16).cuda(), row)
    with pytest.raises(ValueError):
        ops.combine_grad(d, d, row, w, ops.ROUTE_SWITCH)
    with pytest.raises(ValueError):
        ops.combine_grad(d, d, row, w, 0, shared_gate=w[:, 0])
    with pytest.raises(ops._lib.ZmoeError, match="mode"):
        ops.combine_grad(d, d, row, w, 3)


def test_empty_batches():
    ops = _ops()
    z = torch.zeros(0, 16, dtype=torch.bfloat16).cuda()
    row = torch.zeros(0, 4, dtype=torch.int32).cuda()
    assert ops.permute_grad(z, row).shape == (0, 16)
    got = ops.combine_grad(z, z, row, torch.zeros(0, 4).cuda(), 0)
    assert got[0].shape == (0, 16) and got[1].shape == (0, 4)
    # tokens, but none with a row
    row = torch.full((3, 2), -1, dtype=torch.int32).cuda()
    assert (ops.permute_grad(z, row) == 0).all()
    assert (ops.combine_grad(torch.ones(3, 16, dtype=torch.bfloat16).cuda(), z, row, torch.ones(3, 2).cuda(), 0)[1] == 0).all()
    counts, offsets, *_ = ops.permute(row, torch.ones(3, 16, dtype=torch.bfloat16).cuda(), 4)
    assert (counts == 0).all() and (offsets == 0).all()


# lists of 131072 pairs and more: full and ragged last CTAs, one expert, as many as there may be
@pytest.mark.parametrize("T,k,E", [(131072, 1, 1), (131073, 1, 3), (32768, 4, 60), (43692, 3, 700), (17001, 8, 1024), (4229, 31, 896),
                                   (4096, 32, 1024)])
@pytest.mark.parametrize("bad", [False, True])
def test_sort_of_many_pairs(T, k, E, bad):
    ops = _ops()
    k_e = min(k, E)
    idx = np.full((T, k), -1, np.int32)
    idx[:, :k_e] = _idx(T, k_e, E, T, bad)
    offs, tor, row_of = _plain_rows(idx, E)
    x = torch.randn(T, 8, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16)
    for xd in (x.cuda(), None):
        counts, offsets, r_of, t_of, xp = ops.permute(torch.from_numpy(idx).cuda(), xd, E)
        assert np.array_equal(counts.cpu().numpy(), np.diff(offs))
        assert np.array_equal(offsets.cpu().numpy(), offs)
        assert np.array_equal(r_of.cpu().numpy(), row_of)
        assert np.array_equal(t_of[:len(tor)].cpu().numpy(), tor)
        if xd is not None:
            assert torch.equal(xp[:len(tor)].cpu(), x[torch.from_numpy(tor).long()])


def test_sort_of_many_pairs_leaves_rows_behind_the_last():
    from zmoe._lib import PermuteArgs, check, lib
    import ctypes
    T, k, E, H = 80000, 2, 60, 8
    idx = torch.full((T, k), -1, dtype=torch.int32)
    idx[::100, 1] = 7
    n = T // 100
    d, x = idx.cuda(), torch.ones(T, H, dtype=torch.bfloat16).cuda()
    counts, offsets = torch.empty(E, dtype=torch.int32).cuda(), torch.empty(E + 1, dtype=torch.int32).cuda()
    row_of, tor = torch.empty(T, k, dtype=torch.int32).cuda(), torch.full((T * k,), -7, dtype=torch.int32).cuda()
    xp = torch.full((T * k, H), 5.0, dtype=torch.bfloat16).cuda()
    a = PermuteArgs(topk_idx=d.data_ptr(), x=x.data_ptr(), T=T, H=H, E=E, k=k, counts=counts.data_ptr(), offsets=offsets.data_ptr(),
                    row_of=row_of.data_ptr(), token_of_row=tor.data_ptr(), xp=xp.data_ptr())
    check(lib.zmoe_permute(ctypes.byref(a), torch.cuda.current_stream().cuda_stream), "zmoe_permute")
    assert tor[:n].tolist() == list(range(0, T, 100)) and (tor[n:] == -7).all()
    assert (xp[:n] == 1).all() and (xp[n:] == 5).all()
    assert int(counts.sum()) == n and int(counts[7]) == n


@pytest.mark.parametrize("T", [300, 9000, 70000])
def test_sort_replayed_and_on_two_streams(T):
    ops = _ops()
    k, E, H = 2, 60, 64
    idx = [torch.from_numpy(_idx(T, k, E, s)).cuda() for s in range(3)]
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16).cuda()
    want = [ops.permute(i, x, E) for i in idx]
    held = idx[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.permute(held, x, E)
        total = got[4].float().sum(0)                   # reads the copy right behind it
    for i, w in zip(idx, want):
        held.copy_(i)
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(got, w))
        assert torch.equal(total, w[4].float().sum(0))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    res = [[], []]
    torch.cuda.synchronize()
    for _ in range(10):
        for j, q in enumerate(streams):
            with torch.cuda.stream(q):
                res[j].append(ops.permute(idx[j], x, E))
    torch.cuda.synchronize()
    for j in range(2):
        assert all(torch.equal(p, q) for r in res[j] for p, q in zip(r, want[j]))
