"""The sort, the adapters and their gradients together, as a layer uses them:
experts' adapters in training under frozen projections, requests' adapters in
serving beside the shared expert; then the forms a caller may use them in (two
streams at once, a first call inside a graph, long offsets, the error path)."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

from oracle import adapters

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
HALF = 2.0 ** -8                                       # half a step of BF16, relative
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _ops():
    from zmoe import ops
    return ops


def test_training_step_of_expert_adapters():
    """x -> sort -> frozen expert projection + adapter -> weighted return, and
    back to x, the adapters, the weights and the shared gate, against torch's
    differentiation in 64 bits.  Between the kernels values are BF16: each
    rounding is off by at most HALF of its value, carried on by absolute values."""
    ops = _ops()
    T, E, k, H, N, R = 150, 5, 2, 64, 72, 16
    g = torch.Generator().manual_seed(1)
    bf = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(BF)  # noqa: E731
    x, dout, ysh = bf(T, H), bf(T, N), bf(T, N)
    W = bf(E, N, H, std=H ** -0.5)
    a, b = bf(E, R, H, std=H ** -0.5), bf(E, N, R, std=R ** -0.5)
    scale, w, gate = torch.rand(E, generator=g) + 0.5, torch.rand(T, k, generator=g), torch.rand(T, generator=g)
    idx = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).to(torch.int32)
    idx[::7, 1] = -1                                   # slots without a row

    cu = [t.cuda() for t in (x, dout, ysh, a, b, scale, w, gate)]
    xd, doutd, yshd, ad, bd, sd, wd, gated = cu
    counts, offsets, row_of, tor, xp = ops.permute(idx.cuda(), xd, E)
    n = int(offsets[-1])
    expert = torch.repeat_interleave(torch.arange(E), counts.cpu().long())
    Wr = W[expert].cuda().float()                      # frozen projections, by row
    xp = xp[:n].contiguous()
    y0 = torch.bmm(Wr, xp.float()[:, :, None])[:, :, 0].to(BF)
    u = torch.empty(n, R).cuda()
    y = ops.lora(xp, y0, ad, bd, sd, offsets, u=u)
    out = ops.combine(y, row_of, wd, ops.ROUTE_QWEN, yshd, gated)
    dy, dw, dysh, dg, _ = ops.combine_grad(doutd, y, row_of, wd, ops.ROUTE_QWEN, yshd, gated)
    back = torch.bmm(Wr.transpose(1, 2), dy.float()[:, :, None])[:, :, 0].to(BF)
    dxp, da, db = ops.lora_grad(dy, xp, u, ad, bd, sd, offsets, base=back)
    dx = ops.permute_grad(dxp, row_of)

    # 64 bits: M_e = W_e + s_e B_e A_e
    leaves = [t.double().requires_grad_() for t in (x, a, b, w, gate)]
    x6, a6, b6, w6, g6 = leaves
    M = W.double() + scale.double()[:, None, None] * (b6 @ a6)
    keep = (idx >= 0).double()
    yt = torch.einsum("tknh,th->tkn", M[idx.clamp(min=0).long()], x6)
    ref = (yt * (w6 * keep)[:, :, None]).sum(1) + g6[:, None] * ysh.double()
    (ref * dout.double()).sum().backward()
    gx, ga, gb, gw, gg = (t.grad for t in leaves)

    absM = W.double().abs() + scale.double()[:, None, None] * (b.double().abs() @ a.double().abs())
    slack = 1.05                                       # second order and the fp32 sums
    wk = w.double() * keep
    ay = torch.einsum("tknh,th->tkn", absM[idx.clamp(min=0).long()], x.double().abs())
    tol = slack * HALF * ((2 * ay * wk[:, :, None]).sum(1) + ref.detach().abs())
    assert ((out.cpu().double() - ref).abs() <= tol + 1e-6).all()
    # dy = round(w dout); what it loses goes through M to the row, which rounds twice more
    ady = wk[:, :, None] * dout.double().abs()[:, None]
    arow = torch.einsum("tkn,tknh->tkh", ady, absM[idx.clamp(min=0).long()])
    assert ((dx.cpu().double() - gx).abs() <= slack * HALF * (3 * arow.sum(1) + gx.abs()) + 1e-6).all()
    # dw = <dout, y>: y rounds twice (y0, y)
    assert ((dw.cpu().double() - gw * keep).abs() <= slack * HALF * 2 * (ay * dout.double().abs()[:, None]).sum(2) * keep + 1e-6).all()
    assert ((dg.cpu().double() - gg).abs() <= 1e-5 * (1 + (dout.double() * ysh.double()).abs().sum(1))).all()
    assert torch.equal(dysh.cpu(), (gate[:, None] * dout.float()).to(BF))
    # da = sum v^T x with v = s dy B; db = s sum dy^T u: dy and the result round once each
    hot = torch.zeros(T, k, E, dtype=torch.float64).scatter_(2, idx.clamp(min=0).long()[:, :, None], keep[:, :, None])
    s6 = scale.double()
    av = torch.einsum("tkn,tke,enr,e->tker", ady, hot, b.double().abs(), s6)
    assert ((da.cpu().double() - ga).abs() <= slack * HALF * (torch.einsum("tker,th->erh", av, x.double().abs()) + ga.abs()) + 1e-6).all()
    au = torch.einsum("th,erh->ter", x.double().abs(), a.double().abs())
    assert ((db.cpu().double() - gb).abs() <= slack * HALF * (torch.einsum("tkn,tke,ter,e->enr", ady, hot, au, s6) + gb.abs()) + 1e-6).all()


def test_serving_step_beside_the_shared_expert():
    """Adapters of a batch's requests on the shared expert's down projection: the
    plan once, the FFN, then the adapters over its intermediate, in place."""
    ops = _ops()
    T, H, inter, G, R = 40, 256, 128, 4, 8
    g = torch.Generator().manual_seed(2)
    bf = lambda *s, std=0.05: (torch.randn(*s, generator=g) * std).to(BF)  # noqa: E731
    x, mats = bf(T, H, std=1.0), [bf(inter, H), bf(inter, H), bf(H, inter)]
    a, b = bf(G, R, inter, std=inter ** -0.5), bf(G, H, R, std=R ** -0.5)
    ids = torch.tensor([0, 0, 2, -1, 3] * 8, dtype=torch.int32)
    dev = [t.cuda() for t in mats]
    y, h = ops.expert_ffn(x.cuda(), ops.weight_table([dev], "cuda"), None, 1, inter, 0)
    y0 = y.clone()
    offsets, tor = ops.lora_plan(ids.cuda(), G)
    got = ops.lora(h, y, a.cuda(), b.cuda(), None, offsets, tor, out=y)
    assert got is y
    (want, bound), _ = adapters.lora(h.cpu(), y0.cpu(), a, b, None, offsets.cpu(), tor.cpu())
    assert adapters.outside(y, want, bound)[0] == 0
    assert torch.equal(y.cpu()[ids < 0], y0.cpu()[ids < 0])


@pytest.mark.parametrize("T", [64, 900])
def test_two_streams_at_once(T):
    ops = _ops()
    g = torch.Generator().manual_seed(T)
    H, N, G, R = 512, 512, 6, 64
    st, want = [], []
    for i in range(2):
        ids = torch.randint(-1, G, (T,), generator=g, dtype=torch.int32).cuda()
        c = [(torch.randn(*s, generator=g) * 0.1).to(BF).cuda() for s in ((T, H), (T, N), (G, R, H), (G, N, R), (T, N))]
        st.append((ids, *c))

    def step(s):
        ids, x, base, a, b, dy = s
        offsets, tor = ops.lora_plan(ids, G)
        u = torch.zeros(T, R, device="cuda")
        out = ops.lora(x, base, a, b, None, offsets, tor, u=u)
        return (out, u) + ops.lora_grad(dy, x, u, a, b, None, offsets, tor)

    for s in st:
        want.append(step(s))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i, q in enumerate(streams):
            with torch.cuda.stream(q):
                got[i].append(step(st[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(p, q) for p, q in zip(r, want[i]))


def test_first_call_inside_a_graph():
    # a process whose first calls of every entry point are captured
    code = """
import sys; sys.path[:0] = [%r, %r]
import torch
from zmoe import ops
BF = torch.bfloat16
T, E, k, H, N, R = 700, 6, 2, 128, 192, 80
g = torch.Generator().manual_seed(0)
idx = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).to(torch.int32).cuda()
mk = lambda *s: torch.randn(*s, generator=g).to(BF).cuda()
x, a, b, dout = mk(T, H), mk(E, R, H), mk(E, N, R), mk(T, N)
w = torch.rand(T, k, generator=g).cuda()
def step():
    counts, offsets, row_of, tor, xp = ops.permute(idx, x, E)
    u = torch.zeros(T * k, R, device="cuda")
    y = ops.lora(xp, None, a, b, None, offsets, u=u)
    out = ops.combine(y, row_of, w, 0)
    dy, dw, *_ = ops.combine_grad(dout, y, row_of, w, 0)
    dxp, da, db = ops.lora_grad(dy, xp, u, a, b, None, offsets)
    small = ops.lora(xp[:9].contiguous(), None, a, b, None, torch.zeros(E + 1, dtype=torch.int32, device="cuda") + 9)
    return out, dw, da, db, ops.permute_grad(dxp, row_of), small, *ops.lora_plan(idx[:, 0].contiguous(), E)
torch.zeros(1).cuda()
gr = torch.cuda.CUDAGraph()
with torch.cuda.graph(gr):
    held = step()
for _ in range(3): gr.replay()
torch.cuda.synchronize()
again = step()
torch.cuda.synchronize()
assert all(torch.equal(p, q) for p, q in zip(held, again))
print("same")
""" % (ROOT, os.path.join(ROOT, "zipmoe-icml26_b200"))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("same"), r.stderr[-2000:]


def test_offsets_past_32_bits():
    # more than 2^31 elements in the sorted rows, and in an adapter's rows
    ops = _ops()
    T, k, H = 550_001, 2, 2048
    assert T * k * H > 2 ** 31
    idx = torch.tensor([[1, 0]], dtype=torch.int32).repeat(T, 1).cuda()
    x = (torch.arange(T * 8, device="cuda").view(T, 8) % 253).to(BF).repeat(1, H // 8)
    counts, offsets, row_of, tor, xp = ops.permute(idx, x, 2)
    assert offsets.tolist() == [0, T, 2 * T]
    for r, t in ((0, 0), (T - 1, T - 1), (T, 0), (2 * T - 1, T - 1), (2 * T - 5, T - 5)):
        assert torch.equal(xp[r], x[t]) and int(tor[r]) == t
    dx = ops.permute_grad(xp, row_of)
    assert torch.equal(dx[-300:], (x[-300:].float() * 2).to(BF)) and torch.equal(dx[:300], (x[:300].float() * 2).to(BF))
    dy, dw, *_ = ops.combine_grad(x, xp, row_of, torch.full((T, k), 0.5, device="cuda"), 0, dy=xp)
    assert torch.equal(dy[-300:], (x[-300:].float() / 2).to(BF))
    del xp, dx, dy, x
    T, H = 1_100_001, 2048
    x = torch.zeros(T, H, dtype=BF, device="cuda")
    x[-1] = 1
    x[5] = 2
    a, b = torch.full((1, 8, H), 1 / 64, dtype=BF, device="cuda"), torch.full((1, 8, 8), 0.5, dtype=BF, device="cuda")
    offsets = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    u = torch.empty(T, 8, device="cuda")
    out = ops.lora(x, None, a, b, None, offsets, u=u)
    assert (u[-1] == 32).all() and (u[5] == 64).all() and (u[6:-1] == 0).all()
    assert (out[-1] == 128).all() and (out[5] == 256).all() and (out[6:-1] == 0).all()


@pytest.mark.parametrize("R", [16, 104])
def test_wait_timeout_is_reported_and_context_survives(R):
    from zmoe._lib import check, lib

    def error(reset=1):
        code = ctypes.c_int32(-1)
        check(lib.zmoe_kernel_error(ctypes.byref(code), reset), "zmoe_kernel_error")
        return code.value

    ops = _ops()
    T, H, N = 1100, 256, 192
    g = torch.Generator().manual_seed(R)
    mk = lambda *s: (torch.randn(*s, generator=g) * 0.1).to(BF).cuda()  # noqa: E731
    x, a, b, dy, u = mk(T, H), mk(2, R, H), mk(2, N, R), mk(T, N), torch.zeros(T, R, device="cuda")
    offsets = torch.tensor([0, 500, 1000], dtype=torch.int32, device="cuda")
    want = ops.lora(x, None, a, b, None, offsets, u=u), *ops.lora_grad(dy, x, u, a, b, None, offsets)
    torch.cuda.synchronize()
    error()
    assert error() == 0
    for call in (lambda: ops.lora(x, None, a, b, None, offsets), lambda: ops.lora_grad(dy, x, u, a, b, None, offsets)):
        lib.zmoe_debug_ffn_wait(2_000_000, 1)           # clock64 cycles, about 1 ms
        try:
            call()
            torch.cuda.synchronize()
        finally:
            lib.zmoe_debug_ffn_wait(0, 0)
        assert error() == 1
        assert error() == 0
    got = ops.lora(x, None, a, b, None, offsets, u=u), *ops.lora_grad(dy, x, u, a, b, None, offsets)
    torch.cuda.synchronize()
    assert error() == 0
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_token_lists_of_many_rows():
    # 242 thousand tiles, small whole numbers: every sum and output is exact (at most 256)
    ops = _ops()
    T, D, G = 31_000_000, 8, 2
    offsets = torch.tensor([0, 13, T - 5], dtype=torch.int32, device="cuda")
    tor = torch.arange(T - 1, -1, -1, dtype=torch.int32, device="cuda")
    x = (torch.arange(T * D, device="cuda", dtype=torch.int32) % 5).to(BF).view(T, D)
    g = torch.Generator().manual_seed(3)
    a = torch.randint(-1, 2, (G, D, D), generator=g).to(BF).cuda()
    b = torch.eye(D, dtype=BF).flip(0).repeat(G, 1, 1).contiguous().cuda()
    u = torch.zeros(T, D, device="cuda")
    out = ops.lora(x, x, a, b, None, offsets, tor, u=u)
    dx, da, db = ops.lora_grad(x, x, u, a, b, None, offsets, tor)
    for g0, r0, r1 in ((0, 0, 13), (1, 13, T - 5)):
        xr = x[T - r1:T - r0].float()                  # tokens T - 1 - r
        w, bw = a[g0].float(), b[g0].float()
        assert torch.equal(out[T - r1:T - r0].float(), xr + xr @ w.T @ bw.T)
        assert torch.equal(dx[T - r1:T - r0].float(), xr @ bw @ w)
        assert torch.equal(u[r0:r1], (xr @ w.T).flip(0))
    assert torch.equal(out[:5], x[:5]) and not dx[:5].any() and not u[T - 5:].any()
    xr = x[T - 13:].float()
    assert torch.equal(da[0], ((xr @ b[0].float()).T @ xr).to(BF)) and torch.equal(db[0], (xr.T @ (xr @ a[0].float().T)).to(BF))
