"""64-bit statements of the gradients of permute and combine and of the low-rank
adapters (test infrastructure; plain torch on the CPU).

Each returns its result and, beside it, how far a kernel may be off before its
one rounding to the output type: sums of n products in fp32 in any order are
within n * 2^-23 of the sum of the products' absolute values (2^-24 for a
rounded addition, twice that for one that truncates).
"""
import torch

F64 = torch.float64
STEP = 2.0 ** -23
SPLIT = 2.0 ** -16            # what adding up the products of an fp32 factor's BF16 terms (three, exact) may add


def permute_grad(dxp, row_of, base=None):
    T, k = row_of.shape
    d = dxp.to(F64)
    dx = torch.zeros(T, dxp.shape[1], dtype=F64)
    mag = torch.zeros_like(dx)
    for t in range(T):
        for j in range(k):
            if row_of[t, j] >= 0:
                dx[t] += d[row_of[t, j]]
                mag[t] += d[row_of[t, j]].abs()
        if base is not None:
            dx[t] += base[t].to(F64)
            mag[t] += base[t].to(F64).abs()
    return dx, (k + 1) * STEP * mag


def combine(y, row_of, w, switch=False, y_shared=None, gate=None, x=None):
    """Forward, in 64 bits (zmoe_combine without its rounding)."""
    T, k = row_of.shape
    out = torch.zeros(T, y.shape[1], dtype=F64)
    for t in range(T):
        for j in range(k):
            r = int(row_of[t, j])
            if r >= 0:
                out[t] += w[t, j].to(F64) * y[r].to(F64)
            elif switch:
                out[t] += w[t, j].to(F64) * x[t].to(F64)
        if y_shared is not None:
            out[t] += (1.0 if gate is None else gate[t].to(F64)) * y_shared[t].to(F64)
    return out


def combine_grad(dout, y, row_of, w, switch=False, y_shared=None, gate=None, x=None):
    """{name: (value, bound)}; dy rows that no slot names are NaN."""
    T, k = row_of.shape
    H = dout.shape[1]
    d = dout.to(F64)
    dy = torch.full((y.shape[0], H), float("nan"), dtype=F64)
    dw, dwb = torch.zeros(T, k, dtype=F64), torch.zeros(T, k, dtype=F64)
    dx = torch.zeros(T, H, dtype=F64)
    for t in range(T):
        for j in range(k):
            r = int(row_of[t, j])
            if r >= 0:
                dy[r] = w[t, j].to(F64) * d[t]
                p = d[t] * y[r].to(F64)
            elif switch:
                dx[t] = w[t, j].to(F64) * d[t]
                p = d[t] * x[t].to(F64)
            else:
                continue
            dw[t, j], dwb[t, j] = p.sum(), p.abs().sum() * H * STEP
    out = {"dy": (dy, dy.abs() * STEP), "dw": (dw, dwb)}
    if y_shared is not None:
        g = torch.ones(T, dtype=F64) if gate is None else gate.to(F64)
        out["dysh"] = (g[:, None] * d, (g[:, None] * d).abs() * STEP)
        p = d * y_shared.to(F64)
        out["dg"] = (p.sum(1), p.abs().sum(1) * H * STEP)
    if switch:
        out["dx"] = (dx, dx.abs() * STEP)
    return out


def plan(ids, G):
    """offsets [G + 1] and token_of_row [T]; ids outside [0, G) come last."""
    ids = [int(i) if 0 <= int(i) < G else G for i in ids]
    order = [t for g in range(G + 1) for t, i in enumerate(ids) if i == g]
    offsets = [0]
    for g in range(G):
        offsets.append(offsets[-1] + ids.count(g))
    return torch.tensor(offsets, dtype=torch.int32), torch.tensor(order, dtype=torch.int32)


def _groups(offsets, token_of_row, a, b, rank, scale):
    for g in range(a.shape[0]):
        r0, r1 = int(offsets[g]), int(offsets[g + 1])
        rows = torch.arange(r0, r1)
        t = rows if token_of_row is None else token_of_row[rows].long()
        rk = a.shape[1] if rank is None else min(max(int(rank[g]), 0), a.shape[1])
        s = 1.0 if scale is None else float(scale[g])
        yield g, rows, t, a[g, :rk].to(F64), b[g, :, :rk].to(F64), s, rk


def lora(x, base, a, b, scale, offsets, token_of_row=None, rank=None):
    """(out, bound), (u, bound); u rows behind the last adapter are NaN."""
    T, H = x.shape
    G, R, _ = a.shape
    out = torch.zeros(T, b.shape[1], dtype=F64) if base is None else base.to(F64).clone()
    ob = out.abs() * STEP
    u = torch.full((T, R), float("nan"), dtype=F64)
    ub = torch.zeros(T, R, dtype=F64)
    for g, rows, t, A, B, s, rk in _groups(offsets, token_of_row, a, b, rank, scale):
        xt = x[t].to(F64)
        ug = xt @ A.T
        ugb = xt.abs() @ A.abs().T * H * STEP
        u[rows] = 0.0
        u[rows, :rk] = ug
        ub[rows, :rk] = ugb
        out[t] += s * (ug @ B.T)
        ob[t] += abs(s) * (ugb @ B.abs().T + ug.abs() @ B.abs().T * ((R + 4) * STEP + SPLIT))
    return (out, ob + out.abs() * STEP), (u, ub)


def lora_grad(dy, x, u, a, b, scale, offsets, token_of_row=None, rank=None, base=None):
    """{name: (value, bound)} for dx, da, db."""
    T, H = x.shape
    G, R, _ = a.shape
    N = b.shape[1]
    dx = torch.zeros(T, H, dtype=F64) if base is None else base.to(F64).clone()
    dxb = dx.abs() * STEP
    da, dab = torch.zeros(G, R, H, dtype=F64), torch.zeros(G, R, H, dtype=F64)
    db, dbb = torch.zeros(G, N, R, dtype=F64), torch.zeros(G, N, R, dtype=F64)
    for g, rows, t, A, B, s, rk in _groups(offsets, token_of_row, a, b, rank, scale):
        d, xt, n = dy[t].to(F64), x[t].to(F64), len(rows)
        v = s * (d @ B)
        vb = abs(s) * (d.abs() @ B.abs()) * N * STEP + v.abs() * STEP
        dx[t] += v @ A
        dxb[t] += vb @ A.abs() + v.abs() @ A.abs() * ((R + 4) * STEP + SPLIT)
        da[g, :rk] = v.T @ xt
        dab[g, :rk] = vb.T @ xt.abs() + v.abs().T @ xt.abs() * ((n + 4) * STEP + SPLIT)
        ug = u[rows, :rk].to(F64)
        db[g, :, :rk] = s * (d.T @ ug)
        dbb[g, :, :rk] = abs(s) * (d.abs().T @ ug.abs()) * ((n + 4) * STEP + SPLIT)
    return {"dx": (dx, dxb + dx.abs() * STEP), "da": (da, dab), "db": (db, dbb)}


def outside(got, want, bound):
    """Whether a rounded output is further off than half a step of its type and
    the bound before rounding; equal where the value must be."""
    half = torch.finfo(got.dtype).eps / 2
    g = got.cpu().to(F64)
    tol = bound + half * (want.abs() + bound) + torch.finfo(got.dtype).tiny
    bad = ~((g - want).abs() <= tol)
    return int(bad.sum()), float(((g - want).abs() / tol).nan_to_num(float("inf")).max()) if g.numel() else 0.0
