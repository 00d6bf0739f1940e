"""Argument checks of the gradient and adapter entry points, which refuse before
any CUDA call (no GPU needed), and their struct layouts."""
import ctypes
import os
import subprocess
import tempfile

import torch

from oracle import adapters

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 4096                                                # a non-null, aligned pointer that is never followed


def _lib():
    from zmoe import _lib
    return _lib


def _refused(fn, args, text):
    assert fn(ctypes.byref(args), None) == 1
    assert text in _lib().lib.zmoe_last_error(), _lib().lib.zmoe_last_error()


def test_struct_layouts():
    L = _lib()
    names = ["permute_grad", "combine_grad", "lora", "lora_grad"]
    src = ('#include "zmoe.h"\n#include <stdio.h>\nint main(){printf("%zu %zu %zu %zu %d %d", '
           + ", ".join(f"sizeof(zmoe_{n}_args)" for n in names) + ", ZMOE_LORA_MAX_RANK, ZMOE_LORA_ROWS);}")
    with tempfile.TemporaryDirectory() as d:
        open(os.path.join(d, "s.c"), "w").write(src)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", os.path.join(d, "s"), os.path.join(d, "s.c")],
                       check=True)
        got = [int(v) for v in subprocess.run([os.path.join(d, "s")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(c) for c in (L.PermuteGradArgs, L.CombineGradArgs, L.LoraArgs, L.LoraGradArgs)] + [L.LORA_MAX_RANK, L.LORA_ROWS]


def test_permute_grad_refuses():
    L = _lib()
    ok = dict(dxp=P, row_of=P, base=None, T=4, H=16, k=2, rows=8, dx=P)
    for kw, text in (({"H": 12}, b"multiple of 8"), ({"H": 0}, b"multiple of 8"), ({"dx": None}, b"null"),
                     ({"row_of": None}, b"null"), ({"dxp": None}, b"null"), ({"k": 0}, b"k < 1"), ({"T": -1}, b"negative"),
                     ({"dxp": P + 2}, b"aligned"), ({"base": P + 8}, b"aligned")):
        _refused(L.lib.zmoe_permute_grad, L.PermuteGradArgs(**dict(ok, **kw)), text)


def test_combine_grad_refuses():
    L = _lib()
    ok = dict(dout=P, y=P, y_shared=None, shared_gate=None, row_of=P, topk_w=P, x=None, T=4, H=16, k=2, mode=0, rows=8,
              dy=P, dtopk_w=P, dy_shared=None, dshared_gate=None, dx=None)
    for kw, text in (({"mode": 3}, b"mode"), ({"mode": 2, "k": 1}, b"Switch"), ({"dshared_gate": P}, b"y_shared"),
                     ({"H": 20}, b"multiple of 8"), ({"y": None}, b"null"), ({"dy": P + 4}, b"aligned"), ({"k": 0}, b"k < 1")):
        _refused(L.lib.zmoe_combine_grad, L.CombineGradArgs(**dict(ok, **kw)), text)


def test_lora_refuses():
    L = _lib()
    ok = dict(x=P, base=P, a=P, b=P, scale=P, rank=None, offsets=P, token_of_row=None, T=4, H=16, N=16, G=2, R=8, out=P, scratch=P)
    for kw, text in (({"R": 12}, b"R=12"), ({"R": 136}, b"R=136"), ({"R": 0}, b"R=0"), ({"H": 20}, b"H=20"),
                     ({"N": 4}, b"N=4"), ({"G": 0}, b"G < 1"), ({"T": -1}, b"T < 0"), ({"x": None}, b"null"),
                     ({"offsets": None}, b"null"), ({"T": 513, "scratch": None}, b"null"), ({"a": P + 2}, b"aligned"), ({"out": P + 8}, b"aligned"),
                     ({"H": 32776}, b"above")):
        _refused(L.lib.zmoe_lora, L.LoraArgs(**dict(ok, **kw)), text)
    ok = dict(dy=P, x=P, u=P, a=P, b=P, scale=P, rank=None, offsets=P, token_of_row=None, base=None, T=4, H=16, N=16,
              G=2, R=8, dx=P, da=P, db=P, scratch=P)
    for kw, text in (({"da": None}, b"together"), ({"dx": None, "da": None, "db": None}, b"no output"), ({"scratch": None}, b"null"),
                     ({"u": None}, b"null"), ({"R": 12}, b"R=12"), ({"dy": P + 2}, b"aligned"), ({"G": 0}, b"G < 1")):
        _refused(L.lib.zmoe_lora_grad, L.LoraGradArgs(**dict(ok, **kw)), text)
    assert L.lib.zmoe_lora_plan(P, 4, 0, P, P, None) == 1
    assert L.lib.zmoe_lora_plan(None, 4, 3, P, P, None) == 1
    assert L.lib.zmoe_lora_plan(P, 4, 1024, P, P, None) == 1


def test_statements_agree_with_autograd():
    # the 64-bit gradient statements against torch's own differentiation of the
    # forward statements' formulas
    g = torch.Generator().manual_seed(0)
    T, H, N, G, R = 11, 16, 24, 3, 8
    ids = torch.randint(-1, G, (T,), generator=g)
    offsets, tor = adapters.plan(ids, G)
    x, base, dy = (torch.randn(T, n, generator=g).double() for n in (H, N, N))
    a, b, s = torch.randn(G, R, H, generator=g).double(), torch.randn(G, N, R, generator=g).double(), torch.rand(G, generator=g)
    rank = torch.tensor([8, 3, 5])
    keep = (torch.arange(R)[None] < rank[:, None]).double()
    xs, am, bm = (t.clone().requires_grad_() for t in (x, a, b))
    pick = torch.nn.functional.one_hot(torch.where(ids < 0, G, ids).long(), G + 1)[:, :G].double()
    ug = torch.einsum("th,grh->tgr", xs, am * keep[:, :, None])
    out = base + torch.einsum("tgr,gnr,tg->tn", ug, bm * keep[:, None], pick * s.double())
    (want, _), (u, _) = adapters.lora(x, base, a, b, s, offsets, tor, rank)
    assert torch.allclose(out, want)
    (out * dy).sum().backward()
    got = adapters.lora_grad(dy, x, torch.nan_to_num(u), a, b, s, offsets, tor, rank)
    for n, t in (("dx", xs), ("da", am), ("db", bm)):
        assert torch.allclose(got[n][0], t.grad), n


def test_refuses_lengths_and_aliases():
    L = _lib()
    ok = dict(x=P, base=P, a=P, b=P, scale=P, rank=None, offsets=P, token_of_row=None, T=4, H=16, N=16, G=2, R=8, out=P, scratch=P)
    _refused(L.lib.zmoe_lora, L.LoraArgs(**dict(ok, T=2 ** 30 + 1)), b"above")
    Q = 2 * P
    ok = dict(dy=P, x=P, u=P, a=P, b=P, scale=P, rank=None, offsets=P, token_of_row=None, base=None, T=4, H=16, N=16,
              G=2, R=8, dx=Q, da=Q, db=Q, scratch=Q)
    for kw, text in (({"T": 2 ** 30 + 1}, b"above"), ({"dy": Q}, b"must not be"), ({"x": Q}, b"must not be")):
        _refused(L.lib.zmoe_lora_grad, L.LoraGradArgs(**dict(ok, **kw)), text)
    assert L.lib.zmoe_lora_plan(P, 2 ** 31 - 1, 3, P, P, None) == 1
    _refused(L.lib.zmoe_permute, L.PermuteArgs(topk_idx=P, x=None, T=2 ** 31 - 1, H=0, k=1, E=4, capacity=0, seq_len=0,
                                               counts=P, offsets=P, row_of=P, token_of_row=P, xp=None), b"too many")
