"""The sums between an adapter's two products keep all their 24 bits.  Whole
numbers of 20 bits that cancel in the second product down to a few units: every
sum is exact in fp32, so the outputs are, and a factor held in fewer bits shows."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _ops():
    from zmoe import ops
    return ops


def _digits(n, g):
    """n numbers of 20 bits as three BF16 values each, and the sums."""
    d = torch.stack([torch.randint(64, 128, (n,), generator=g) * 2 ** 13, torch.randint(64, 128, (n,), generator=g) * 2 ** 6,
                     torch.randint(0, 64, (n,), generator=g)], 1)
    return d, d.sum(1)


def _case(T, R):
    g = torch.Generator().manual_seed(T + R)
    G, H, N = 2, 264, 200
    cut = T // 2 + 1
    offsets = torch.tensor([0, cut, T], dtype=torch.int32)
    tor = torch.arange(T - 1, -1, -1, dtype=torch.int32)
    scale = torch.tensor([2.0, 0.5])
    group = torch.empty(T, dtype=torch.long)
    group[tor[:cut].long()], group[tor[cut:].long()] = 0, 1
    d, total = _digits(T, g)
    small = 2 * torch.randint(-8, 9, (T,), generator=g)
    return g, G, H, N, offsets, tor, scale, group, d, total, small


SIZES = [(5, 16), (5, 64), (5, 104), (300, 40), (1300, 16), (1300, 64), (1300, 104)]


@pytest.mark.parametrize("T,R", SIZES)
def test_forward(T, R):
    g, G, H, N, offsets, tor, scale, group, d, total, small = _case(T, R)
    r0, r1 = 3, R - 2
    x = torch.randint(-3, 4, (T, H), generator=g)
    x[:, :3], x[:, 3] = d, small
    a, b = torch.zeros(G, R, H), torch.zeros(G, N, R)
    a[:, :, :3], a[:, r0, 3] = 1, 1
    b[:, :, r0], b[:, :, r1] = 1, -1
    base = torch.randint(-9, 10, (T, N), generator=g).to(BF)
    u = torch.empty(T, R).cuda()
    out = _ops().lora(x.to(BF).cuda(), base.cuda(), a.to(BF).cuda(), b.to(BF).cuda(), scale.cuda(), offsets.cuda(),
                      tor.cuda(), u=u)
    want = total[:, None].repeat(1, R)
    want[:, r0] += small
    assert torch.equal(u.cpu(), want.flip(0).float())
    assert torch.equal(out.cpu(), (base.float() + (scale[group] * small)[:, None]).to(BF))


@pytest.mark.parametrize("T,R", SIZES)
def test_gradient_of_x_and_of_a(T, R):
    g, G, H, N, offsets, tor, scale, group, d, total, small = _case(T, R)
    r0, r1 = 3, R - 2
    # a pair of tokens in each group with the same large number and x of opposite signs
    first = [int(torch.nonzero(group == e)[0]) for e in range(G)]
    last = [int(torch.nonzero(group == e)[-1]) for e in range(G)]
    x = torch.zeros(T, H)
    beta = torch.randint(-1, 2, (H,), generator=g).float()
    for i, j in zip(first, last):
        d[j] = d[i]
        x[i], x[j] = beta, -beta
    dy = torch.zeros(T, N)
    dy[:, :3], dy[:, 3] = d.float(), small.float()
    a, b = torch.zeros(G, R, H), torch.zeros(G, N, R)
    b[:, :3], b[:, 3, r0] = 1, 1
    alpha = torch.randint(-1, 2, (G, H), generator=g).float()
    a[:, r0], a[:, r1] = alpha, -alpha
    base = torch.randint(-9, 10, (T, H), generator=g).to(BF)
    dx, da, _ = _ops().lora_grad(dy.to(BF).cuda(), x.to(BF).cuda(), torch.zeros(T, R).cuda(), a.to(BF).cuda(), b.to(BF).cuda(),
                                 scale.cuda(), offsets.cuda(), tor.cuda(), base=base.cuda())
    assert torch.equal(dx.cpu(), (base.float() + (scale[group] * small)[:, None] * alpha[group]).to(BF))
    want = torch.zeros(G, R, H)
    for e in range(G):
        want[e, r0] = scale[e] * (small[first[e]] - small[last[e]]) * beta
    assert torch.equal(da.cpu(), want.to(BF))


@pytest.mark.parametrize("T,R", SIZES)
def test_gradient_of_b(T, R):
    g, G, H, N, offsets, tor, scale, group, d, total, small = _case(T, R)
    row = torch.empty(T, dtype=torch.long)
    row[tor.long()] = torch.arange(T)
    dy, u, want = torch.zeros(T, N), torch.zeros(T, R), torch.zeros(G, N, R)
    for e in range(G):
        i, j = int(torch.nonzero(group == e)[0]), int(torch.nonzero(group == e)[-1])
        beta = torch.randint(-1, 2, (N,), generator=g).float()
        big, unit = _digits(R, g)[1], 2 * torch.randint(-60, 61, (R,), generator=g)
        dy[i], dy[j] = beta, -beta
        u[row[i]], u[row[j]] = (big + unit).float(), big.float()
        want[e] = scale[e] * beta[:, None] * unit
    a, b = torch.zeros(G, R, H, dtype=BF), torch.zeros(G, N, R, dtype=BF)
    _, _, db = _ops().lora_grad(dy.to(BF).cuda(), torch.zeros(T, H, dtype=BF).cuda(), u.cuda(), a.cuda(), b.cuda(),
                                scale.cuda(), offsets.cuda(), tor.cuda())
    assert torch.equal(db.cpu(), want.to(BF))
