"""Outputs in the place of their own operand, as the header allows, and the
refusals of the wrappers."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _ops():
    from zmoe import ops
    return ops


def _grad(p):
    import ctypes
    from zmoe._lib import check, lib
    check(lib.zmoe_combine_grad(ctypes.byref(p), torch.cuda.current_stream().cuda_stream), "zmoe_combine_grad")


@pytest.mark.parametrize("switch", [False, True])
def test_combine_grad_in_place(switch):
    from zmoe._lib import CombineGradArgs
    ops = _ops()
    g = torch.Generator().manual_seed(1)
    T, k, E, H = 70, 1 if switch else 3, 6, 264
    idx = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).to(torch.int32)
    idx[::5, 0] = -1
    mk = lambda *s: torch.randn(*s, generator=g).to(BF).cuda()  # noqa: E731
    dout, ysh, x, y = mk(T, H), mk(T, H), mk(T, H), mk(T * k, H)
    w, gate = torch.rand(T, k, generator=g).cuda(), torch.rand(T, generator=g).cuda()
    _, _, row_of, _, _ = ops.permute(idx.cuda(), None, E)
    mode = ops.ROUTE_SWITCH if switch else ops.ROUTE_QWEN
    more = dict(x=x) if switch else dict(y_shared=ysh, shared_gate=gate)
    want = ops.combine_grad(dout, y, row_of, w, mode, dy=y.clone(), **more)
    y2, w2, ysh2, gate2, x2 = (t.clone() for t in (y, w, ysh, gate, x))
    p = CombineGradArgs(dout=dout.data_ptr(), y=y2.data_ptr(), row_of=row_of.data_ptr(), topk_w=w2.data_ptr(), T=T, H=H, k=k,
                        mode=mode, rows=T * k, dy=y2.data_ptr(), dtopk_w=w2.data_ptr())
    if switch:
        p.x, p.dx = x2.data_ptr(), x2.data_ptr()
    else:
        p.y_shared = p.dy_shared = ysh2.data_ptr()
        p.shared_gate = p.dshared_gate = gate2.data_ptr()
    _grad(p)
    got = (y2, w2, None, None, x2) if switch else (y2, w2, ysh2, gate2, None)
    for a, b in zip(want, got):
        assert (a is None) == (b is None) and (a is None or torch.equal(a, b))


def test_wrappers_refuse_overlap():
    ops = _ops()
    T, H, G, R = 40, 64, 2, 8
    buf = torch.zeros(T + 1, H, dtype=BF).cuda()
    x, shifted = buf[:T], buf[1:]
    a, b = torch.zeros(G, R, H, dtype=BF).cuda(), torch.zeros(G, H, R, dtype=BF).cuda()
    offsets, u = torch.tensor([0, 9, T], dtype=torch.int32).cuda(), torch.zeros(T, R).cuda()
    row_of = torch.arange(T, dtype=torch.int32).cuda()[:, None]
    err = ops._lib.ZmoeError
    for call in (lambda: ops.lora(x, None, a, b, None, offsets, out=x), lambda: ops.lora(x, x, a, b, None, offsets, out=x),
                 lambda: ops.lora(x.clone(), x, a, b, None, offsets, out=shifted),
                 lambda: ops.lora_grad(x, x.clone(), u, a, b, None, offsets, dx=shifted),
                 lambda: ops.permute_grad(x, row_of, dx=x), lambda: ops.permute_grad(x.clone(), row_of, base=x, dx=shifted),
                 lambda: ops.combine_grad(x, x.clone(), row_of, torch.ones(T, 1).cuda(), 0, dy=x)):
        with pytest.raises(err, match="overlap"):
            call()
