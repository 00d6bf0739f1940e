"""Low-rank adapters of many requests and their gradient against 64-bit
statements, with the bounds derived there."""
import pytest
import torch

from oracle import adapters

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _ops():
    from zmoe import ops
    return ops


def _cu(t):
    return None if t is None else t.cuda()


def _ids(kind, T, G, g):
    if kind == "one":
        return torch.zeros(T, dtype=torch.int32)
    if kind == "none":
        return torch.full((T,), -1, dtype=torch.int32)
    if kind == "runs":                                  # requests of some length each
        cut = torch.randint(0, G + 1, (max(1, T // 5),), generator=g)
        ids = cut.repeat_interleave(5)
        return torch.cat([ids, ids[:1].repeat(T)])[:T].to(torch.int32)
    return torch.randint(-1, G + 1, (T,), generator=g, dtype=torch.int32)   # mixed: -1 and G have no adapter


def _case(T, H, N, G, R, kind, seed=0, mixed=True):
    g = torch.Generator().manual_seed(seed * 7919 + T * 31 + H + N + R)
    ids = _ids(kind, T, G, g)
    offsets, tor = adapters.plan(ids, G)
    rank = torch.randint(0, R + 1, (G,), generator=g, dtype=torch.int32) if mixed else None
    a = (torch.randn(G, R, H, generator=g) * H ** -0.5).to(BF)
    b = (torch.randn(G, N, R, generator=g) * R ** -0.5).to(BF)
    if mixed:                                           # what lies behind the rank must not matter
        rank[0] = R
        for e in range(G):
            a[e, int(rank[e]):] = float("nan")
            b[e, :, int(rank[e]):] = float("inf")
    return {"ids": ids, "offsets": offsets, "tor": tor, "rank": rank, "a": a, "b": b,
            "scale": torch.rand(G, generator=g) + 0.5, "x": torch.randn(T, H, generator=g).to(BF),
            "base": torch.randn(T, N, generator=g).to(BF), "dy": torch.randn(T, N, generator=g).to(BF),
            "dx0": torch.randn(T, H, generator=g).to(BF), "gen": g}


SHAPES = [  # T, H, N, G, R, ids
    (1, 8, 8, 1, 8, "one"), (1, 2048, 2048, 8, 16, "mixed"), (7, 72, 136, 3, 24, "mixed"), (8, 256, 264, 1, 8, "one"),
    (9, 2048, 1408, 2, 64, "one"), (33, 520, 8, 40, 16, "mixed"), (64, 1024, 2056, 64, 32, "mixed"),
    (130, 264, 72, 2, 128, "runs"), (127, 64, 64, 1, 16, "one"), (128, 64, 128, 1, 16, "one"), (129, 128, 64, 1, 16, "one"),
    (700, 2048, 1000, 5, 64, "runs"), (1100, 200, 328, 3, 40, "runs"), (1025, 1032, 520, 70, 48, "mixed"),
    (600, 512, 256, 4, 104, "runs"), (20, 64, 64, 3, 16, "none"), (300, 64, 192, 3, 16, "none"),
    (2300, 320, 192, 300, 8, "mixed"),
]


@pytest.mark.parametrize("T,H,N,G,R,kind", SHAPES)
def test_plan(T, H, N, G, R, kind):
    c = _case(T, H, N, G, R, kind)
    offsets, tor = _ops().lora_plan(c["ids"].cuda(), G)
    assert torch.equal(offsets.cpu(), c["offsets"]) and torch.equal(tor.cpu(), c["tor"])


def test_plan_long_and_empty():
    ops = _ops()
    ids = torch.randint(-1, 65, (70001,), dtype=torch.int32, generator=torch.Generator().manual_seed(3))
    offsets, tor = ops.lora_plan(ids.cuda(), 64)
    key = torch.where((ids < 0) | (ids >= 64), 64, ids)
    assert torch.equal(tor.cpu(), torch.argsort(key, stable=True).to(torch.int32))
    assert torch.equal(offsets.cpu(), torch.cat([torch.zeros(1, dtype=torch.long), torch.bincount(key, minlength=65)[:64].cumsum(0)]).int())
    offsets, tor = ops.lora_plan(ids[:0].cuda(), 5)
    assert offsets.tolist() == [0] * 6 and tor.numel() == 0


@pytest.mark.parametrize("T,H,N,G,R,kind", SHAPES)
@pytest.mark.parametrize("form", ["full", "plain ranks", "no base", "in place", "sorted rows"])
def test_lora(T, H, N, G, R, kind, form):
    ops = _ops()
    c = _case(T, H, N, G, R, kind, mixed=form != "plain ranks")
    base = None if form == "no base" else c["base"]
    tor = None if form == "sorted rows" else c["tor"]
    scale = None if form == "plain ranks" else c["scale"]
    bd = _cu(base)
    u = torch.full((T, R), -3.0).cuda()
    out = ops.lora(c["x"].cuda(), bd, c["a"].cuda(), c["b"].cuda(), _cu(scale), c["offsets"].cuda(), _cu(tor),
                   _cu(c["rank"]), out=bd if form == "in place" else None, u=u)
    (want, bound), (uw, ub) = adapters.lora(c["x"], base, c["a"], c["b"], scale, c["offsets"], tor, c["rank"])
    assert adapters.outside(out, want, bound)[0] == 0
    n = int(c["offsets"][-1])
    assert (u[n:] == -3).all()
    assert adapters.outside(u[:n], uw[:n], ub[:n])[0] == 0
    alone = torch.ones(T, dtype=torch.bool)
    alone[torch.arange(n) if tor is None else tor[:n].long()] = False
    if base is not None:                                # tokens without adapter: the same bits
        assert torch.equal(out.cpu()[alone], base[alone])


@pytest.mark.parametrize("T,H,N,G,R,kind", SHAPES)
@pytest.mark.parametrize("form", ["full", "plain ranks", "no base", "in place", "sorted rows"])
def test_lora_grad(T, H, N, G, R, kind, form):
    ops = _ops()
    c = _case(T, H, N, G, R, kind, seed=1, mixed=form != "plain ranks")
    base = None if form == "no base" else c["dx0"]
    tor = None if form == "sorted rows" else c["tor"]
    scale = None if form == "plain ranks" else c["scale"]
    _, (uw, _) = adapters.lora(c["x"], None, c["a"], c["b"], scale, c["offsets"], tor, c["rank"])
    u = uw.float()                                      # NaN behind the last adapter's rows: not read
    bd = _cu(base)
    dx, da, db = ops.lora_grad(c["dy"].cuda(), c["x"].cuda(), u.cuda(), c["a"].cuda(), c["b"].cuda(), _cu(scale),
                               c["offsets"].cuda(), _cu(tor), _cu(c["rank"]), base=bd,
                               dx=bd if form == "in place" else None)
    want = adapters.lora_grad(c["dy"], c["x"], u, c["a"], c["b"], scale, c["offsets"], tor, c["rank"], base)
    for n, got in (("dx", dx), ("da", da), ("db", db)):
        assert adapters.outside(got, *want[n])[0] == 0, n


def test_lora_grad_against_differences():
    # the output is linear in x, in a and in b, each alone: central differences
    # of the 64-bit statement are exact up to their own rounding
    ops = _ops()
    c = _case(150, 72, 80, 3, 16, "runs", mixed=False)
    cu = {n: _cu(t) for n, t in c.items() if torch.is_tensor(t)}
    u = torch.empty(150, 16).cuda()
    ops.lora(cu["x"], cu["base"], cu["a"], cu["b"], cu["scale"], cu["offsets"], cu["tor"], u=u)
    dx, da, db = ops.lora_grad(cu["dy"], cu["x"], u, cu["a"], cu["b"], cu["scale"], cu["offsets"], cu["tor"])
    n = int(c["offsets"][-1])
    uc = u.cpu()
    uc[n:] = 0
    want = adapters.lora_grad(c["dy"], c["x"], uc, c["a"], c["b"], c["scale"], c["offsets"], c["tor"])
    # db is stated from the kernel's own u, which is within its bound of x a^T
    (_, _), (_, ub) = adapters.lora(c["x"], None, c["a"], c["b"], c["scale"], c["offsets"], c["tor"])
    loss = lambda x, a, b: (adapters.lora(x, None, a, b, c["scale"], c["offsets"], c["tor"])[0][0] * c["dy"].double()).sum()  # noqa: E731
    args = [c["x"].double(), c["a"].double(), c["b"].double()]
    for i, (got, name) in enumerate(((dx, "dx"), (da, "da"), (db, "db"))):
        d = torch.randn(args[i].shape, generator=c["gen"], dtype=torch.float64)
        hi, lo = list(args), list(args)
        hi[i], lo[i] = args[i] + d, args[i] - d
        num = (loss(*hi) - loss(*lo)) / 2
        tol = ((want[name][1] * 2 + 2.0 ** -8 * want[name][0].abs()) * d.abs()).sum() + 1e-9
        if name == "db":
            _, slack = zip(*[(g, float((c["dy"][c["tor"][r0:r1].long()].double().abs().T @ ub[r0:r1]).max() * s))
                             for g, (r0, r1, s) in enumerate(zip(c["offsets"], c["offsets"][1:], c["scale"]))])
            tol = tol + sum(s * float(d[g].abs().sum()) for g, s in enumerate(slack))
        assert abs((got.cpu().double() * d).sum() - num) <= tol, name


@pytest.mark.parametrize("T", [5, 700])
def test_lora_same_bits_again_on_another_stream_and_in_a_graph(T):
    ops = _ops()
    c = {n: _cu(t) for n, t in _case(T, 512, 264, 6, 32, "mixed").items() if torch.is_tensor(t)}

    def step():
        u = torch.zeros(T, 32, device="cuda")
        offsets, tor = ops.lora_plan(c["ids"], 6)
        out = ops.lora(c["x"], c["base"], c["a"], c["b"], c["scale"], offsets, tor, c["rank"], u=u)
        return (out, u) + ops.lora_grad(c["dy"], c["x"], u, c["a"], c["b"], c["scale"], offsets, tor, c["rank"],
                                        base=c["dx0"])

    first = step()
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    with torch.cuda.stream(other):
        again = step()
    other.synchronize()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    held = []
    for gr in graphs:
        with torch.cuda.graph(gr):
            held.append(step())
    for gr in graphs + graphs:
        gr.replay()
    torch.cuda.synchronize()
    for got in (again, *held):
        assert all(torch.equal(p, q) for p, q in zip(first, got))


def test_lora_refuses():
    ops = _ops()
    c = {n: _cu(t) for n, t in _case(9, 64, 72, 3, 16, "mixed", mixed=False).items() if torch.is_tensor(t)}

    def call(**kw):
        v = dict(c, **kw)
        return ops.lora(v["x"], v["base"], v["a"], v["b"], v["scale"], v["offsets"], v["tor"], v["rank"])

    c["rank"] = None
    call()
    for kw in ({"x": c["x"].float()}, {"x": c["x"][:, :32]}, {"base": c["base"][:5]}, {"a": c["a"].cpu()},
               {"b": c["b"].transpose(1, 2)}, {"offsets": c["offsets"][:-1]}, {"tor": c["tor"].long()},
               {"scale": c["scale"].double()}, {"rank": torch.zeros(2, dtype=torch.int32).cuda()}):
        with pytest.raises(ValueError):
            call(**kw)
    big = torch.zeros(3, 136, 64, dtype=BF).cuda()
    with pytest.raises(ops._lib.ZmoeError, match="multiple of 8 in"):
        call(a=big, b=torch.zeros(3, 72, 136, dtype=BF).cuda())
    with pytest.raises(ops._lib.ZmoeError, match="G="):
        ops.lora_plan(c["ids"], 0)


def test_lora_empty_batch():
    ops = _ops()
    c = {n: _cu(t) for n, t in _case(4, 64, 72, 3, 16, "mixed", mixed=False).items() if torch.is_tensor(t)}
    offsets, tor = ops.lora_plan(c["ids"][:0], 3)
    z = torch.zeros(0, 16).cuda()
    out = ops.lora(c["x"][:0], c["base"][:0], c["a"], c["b"], c["scale"], offsets, tor, u=z)
    assert out.shape == (0, 72)
    dx, da, db = ops.lora_grad(c["dy"][:0], c["x"][:0], z, c["a"], c["b"], c["scale"], offsets, tor)
    assert dx.shape == (0, 64) and (da == 0).all() and (db == 0).all()
