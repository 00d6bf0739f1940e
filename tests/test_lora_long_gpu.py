"""The tile kernels of the adapters in their steady state: more steps than the
rings of shared memory and TMEM hold, ranks above 64, and dA and dB summed over
clusters of 2 to 8 CTAs.  Against the 64-bit statements and their bounds,
evaluated on the GPU."""
import pytest
import torch

from oracle import adapters

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _ops():
    from zmoe import ops
    return ops


def _case(T, H, N, G, R, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + T + R)
    mk = lambda *s, std=1.0: (torch.randn(*s, generator=g, device="cuda") * std).to(BF)  # noqa: E731
    ends = torch.sort(torch.randint(0, T + 1, (G - 1,), generator=g, device="cuda")).values
    # the last tokens have no adapter
    offsets = torch.cat([torch.zeros(1, device="cuda"), ends.clamp(max=T - 3), torch.tensor([T - 3.0], device="cuda")]).to(torch.int32)
    return {"x": mk(T, H), "dy": mk(T, N), "a": mk(G, R, H, std=H ** -0.5), "b": mk(G, N, R, std=R ** -0.5),
            "scale": torch.rand(G, generator=g, device="cuda") + 0.5, "offsets": offsets,
            "tor": torch.randperm(T, generator=g, device="cuda").to(torch.int32),
            "rank": torch.randint(R - 9, R + 1, (G,), generator=g, device="cuda", dtype=torch.int32),
            "base": mk(T, N), "dx0": mk(T, H)}


def _check(got, pair, name):
    want, bound = pair
    bad, worst = adapters.outside(got.cpu(), want.cpu(), bound.cpu())
    assert bad == 0, (name, bad, worst)


@pytest.mark.parametrize("T,H,N,G,R", [(8000, 2048, 2048, 5, 64), (8000, 2048, 2048, 5, 128), (4000, 5632, 1032, 1, 16),
                                       (1300, 1408, 8200, 2, 104), (8191, 264, 2056, 3, 32)])
def test_forward(T, H, N, G, R):
    c = _case(T, H, N, G, R)
    u = torch.full((T, R), -3.0, device="cuda")
    out = _ops().lora(c["x"], c["base"], c["a"], c["b"], c["scale"], c["offsets"], c["tor"], c["rank"], u=u)
    with torch.device("cuda"):
        ref, (uw, ub) = adapters.lora(c["x"], c["base"], c["a"], c["b"], c["scale"], c["offsets"], c["tor"], c["rank"])
    _check(out, ref, "out")
    n = T - 3
    _check(u[:n], (uw[:n], ub[:n]), "u")
    assert (u[n:] == -3).all()


# (CTAs that share a tile of dA and dB: 4, 4, 8, 8, 8, 8, 2, 4, 1)
@pytest.mark.parametrize("T,H,N,G,R", [(2047, 5632, 2048, 1, 16), (2047, 5632, 2048, 1, 128), (6000, 520, 264, 1, 16),
                                       (6000, 2048, 2048, 1, 128), (6000, 256, 256, 2, 104), (6000, 256, 200, 2, 48),
                                       (1500, 520, 8192, 3, 104), (3000, 1032, 1032, 3, 24), (2500, 1408, 2048, 30, 72)])
def test_gradient(T, H, N, G, R):
    c = _case(T, H, N, G, R, seed=1)
    with torch.device("cuda"):
        _, (uw, _) = adapters.lora(c["x"], None, c["a"], c["b"], c["scale"], c["offsets"], c["tor"], c["rank"])
    u = uw.float()                                      # NaN behind the last adapter's rows: not read
    dx, da, db = _ops().lora_grad(c["dy"], c["x"], u, c["a"], c["b"], c["scale"], c["offsets"], c["tor"], c["rank"], base=c["dx0"])
    with torch.device("cuda"):
        ref = adapters.lora_grad(c["dy"], c["x"], u, c["a"], c["b"], c["scale"], c["offsets"], c["tor"], c["rank"], c["dx0"])
    for name, got in (("dx", dx), ("da", da), ("db", db)):
        _check(got, ref[name], name)


@pytest.mark.parametrize("R", [8, 72])
def test_sums_over_clusters_are_exact(R):
    # whole numbers: every sum is below 2^24, so dA and dB are their exact values, rounded once
    T, D, G = 40_000, 64, 2
    g = torch.Generator(device="cuda").manual_seed(R)
    r = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, device="cuda").float()  # noqa: E731
    x, dy, u, b = r(-2, 3, T, D), r(-2, 3, T, D), r(-9, 10, T, R), torch.zeros(G, D, R, device="cuda")
    b[:, :8, :8] = torch.eye(8, device="cuda")
    offsets = torch.tensor([0, 13, T - 5], dtype=torch.int32, device="cuda")
    a = torch.zeros(G, R, D, device="cuda")
    dx, da, db = _ops().lora_grad(dy.to(BF), x.to(BF), u, a.to(BF), b.to(BF), None, offsets)
    assert not dx.any()
    for e, (r0, r1) in enumerate(((0, 13), (13, T - 5))):
        v = dy[r0:r1].double() @ b[e].double()
        assert torch.equal(da[e], (v.T @ x[r0:r1].double()).to(BF))
        assert torch.equal(db[e], (dy[r0:r1].double().T @ u[r0:r1].double()).to(BF))


@pytest.mark.parametrize("active", [0, 17, 63])
def test_one_adapter_of_a_bank(active):
    # all rows belong to one of 64 adapters: the others' gradients are zeros
    T, H, N, G, R = 3000, 520, 264, 64, 16
    c = _case(T, H, N, G, R, seed=2)
    ids = torch.full((T,), active, dtype=torch.int32, device="cuda")
    offsets, tor = _ops().lora_plan(ids, G)
    u = torch.empty(T, R, device="cuda")
    out = _ops().lora(c["x"], c["base"], c["a"], c["b"], None, offsets, tor, u=u)
    dx, da, db = _ops().lora_grad(c["dy"], c["x"], u, c["a"], c["b"], None, offsets, tor)
    with torch.device("cuda"):
        ref, _ = adapters.lora(c["x"], c["base"], c["a"], c["b"], None, offsets, tor)
        back = adapters.lora_grad(c["dy"], c["x"], u, c["a"], c["b"], None, offsets, tor)
    _check(out, ref, "out")
    for name, got in (("dx", dx), ("da", da), ("db", db)):
        _check(got, back[name], name)
