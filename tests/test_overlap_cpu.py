"""Outputs that overlap what a call still reads are refused (before any CUDA
call, so no GPU is needed); those that may take an operand's place are not."""
import ctypes

MB = 1 << 20


def _lib():
    from zmoe import _lib
    return _lib


def _place(names, **kw):
    """A megabyte of its own for each pointer (never followed)."""
    at = {n: (i + 16) * MB for i, n in enumerate(names)}
    at.update(kw)
    return at


def _refused(fn, args, *names):
    assert fn(ctypes.byref(args), None) == 1
    text = _lib().lib.zmoe_last_error().decode()
    assert "overlap" in text and all(n in text for n in names), text


def test_permute_grad():
    L = _lib()
    p = _place(["dxp", "row_of", "base", "dx"], T=4, H=16, k=2, rows=8)
    call = lambda **kw: (L.lib.zmoe_permute_grad, L.PermuteGradArgs(**dict(p, **kw)))  # noqa: E731
    _refused(*call(dx=p["dxp"]), "dx", "dxp")
    _refused(*call(dx=p["dxp"] + 7 * 32), "dx", "dxp")
    _refused(*call(dx=p["base"] + 32), "dx", "base")
    _refused(*call(dx=p["base"] - 3 * 32), "dx", "base")


def test_combine_grad():
    L = _lib()
    names = ["dout", "y", "y_shared", "shared_gate", "row_of", "topk_w", "dy", "dtopk_w", "dy_shared", "dshared_gate"]
    p = _place(names, T=4, H=16, k=2, rows=8, mode=0, x=None, dx=None)
    call = lambda **kw: (L.lib.zmoe_combine_grad, L.CombineGradArgs(**dict(p, **kw)))  # noqa: E731
    _refused(*call(dy=p["dout"]), "dy", "dout")
    _refused(*call(dy=p["y"] + 32), "dy", "y")
    _refused(*call(dy_shared=p["dout"]), "dy_shared", "dout")
    _refused(*call(dy_shared=p["dy"] + 7 * 32), "dy_shared", "dy")
    _refused(*call(dtopk_w=p["row_of"]), "dtopk_w", "row_of")
    _refused(*call(dshared_gate=p["topk_w"]), "dshared_gate", "topk_w")


def test_lora():
    L = _lib()
    p = _place(["x", "base", "a", "b", "scale", "rank", "offsets", "token_of_row", "out", "u", "scratch"], T=600, H=16, N=16, G=2, R=8)
    call = lambda **kw: (L.lib.zmoe_lora, L.LoraArgs(**dict(p, **kw)))  # noqa: E731
    _refused(*call(out=p["x"]), "out", "x")
    _refused(*call(out=p["x"], base=p["x"]), "out", "x")
    _refused(*call(out=p["base"] + 32), "out", "base")
    _refused(*call(u=p["out"] + 32), "u", "out")
    _refused(*call(u=p["scratch"]), "scratch", "u")
    _refused(*call(out=p["a"]), "out", "a")


def test_lora_grad():
    L = _lib()
    names = ["dy", "x", "u", "a", "b", "scale", "rank", "offsets", "token_of_row", "base", "dx", "da", "db", "scratch"]
    p = _place(names, T=600, H=16, N=16, G=2, R=8)
    call = lambda **kw: (L.lib.zmoe_lora_grad, L.LoraGradArgs(**dict(p, **kw)))  # noqa: E731
    _refused(*call(dx=p["dy"] + 32), "dx", "dy")
    _refused(*call(dx=p["x"] - 32), "dx", "x")
    _refused(*call(dx=p["base"] + 32), "dx", "base")
    _refused(*call(da=p["a"]), "da", "a")
    _refused(*call(db=p["da"]), "db", "da")
    _refused(*call(scratch=p["u"]), "scratch", "u")
    _refused(*call(da=None, db=None, dx=p["dy"], base=p["dy"] + 32), "dx", "base")


def test_lora_plan():
    L = _lib()
    for off, tor in ((1 * MB, 2 * MB), (2 * MB, 3 * MB), (3 * MB, 3 * MB + 8)):
        assert L.lib.zmoe_lora_plan(2 * MB if tor != 3 * MB + 8 else MB, 100, 5, off, tor, None) == 1
        assert b"overlap" in L.lib.zmoe_last_error()
