"""Timed operators: tokens sorted by expert and sent back with their weights,
the gradients of both, and low-rank adapters beside a shared projection with
their gradient.

``listed()`` and ``draw()`` give cases, ``prepare()`` a case's inputs,
``run()`` one pass: through the framework's entry points where ``own`` is true,
in plain torch operations where it is false.  ``exact()`` is the same result in
64 bits, written apart from the plain form.
"""
import math
import os
import sys

import torch

own = False

ROUTE_QWEN, ROUTE_DEEPSEEK, ROUTE_SWITCH = 0, 1, 2


def _ops():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "zipmoe-icml26_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from zmoe import ops
    return ops


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one decoded token through a 60-expert top-4 layer
        {"name": "sort-decode", "op": "sort", "T": 1, "E": 60, "k": 4, "H": 2048},
        # a training batch through a 64-expert top-6 layer, one token short of a round length
        {"name": "sort-train", "op": "sort", "T": 16383, "E": 64, "k": 6, "H": 2048},
        # gradient of the sort for one short sequence, alone
        {"name": "sort-grad-short", "op": "sort_grad", "T": 509, "E": 60, "k": 4, "H": 2048, "base": False},
        # the same for a training batch, added to the gradient that came through the shared expert
        {"name": "sort-grad-train", "op": "sort_grad", "T": 16383, "E": 64, "k": 6, "H": 2048, "base": True},
        # weighted return, top-4 with the gated shared expert: the layer's usual step
        {"name": "combine-grad-gated", "op": "combine_grad", "T": 512, "E": 60, "k": 4, "H": 2048, "mode": ROUTE_QWEN,
         "shared": True, "gate": True, "capacity": 0, "seq": 0},
        # top-1 with a capacity: dropped tokens pass through
        {"name": "combine-grad-capacity", "op": "combine_grad", "T": 4096, "E": 128, "k": 1, "H": 1024,
         "mode": ROUTE_SWITCH, "shared": False, "gate": False, "capacity": 40, "seq": 512},
        # top-6 with an ungated shared expert, a training batch
        {"name": "combine-grad-train", "op": "combine_grad", "T": 16383, "E": 64, "k": 6, "H": 2048,
         "mode": ROUTE_DEEPSEEK, "shared": True, "gate": False, "capacity": 0, "seq": 0},
        # one request decoding with its adapter
        {"name": "lora-decode-1", "op": "lora", "T": 1, "requests": 1, "G": 8, "R": 16, "H": 2048, "N": 2048,
         "mixed": False, "rows": "requests"},
        # many requests decoding at once, adapters of several ranks, a few requests with none
        {"name": "lora-decode-96", "op": "lora", "T": 96, "requests": 96, "G": 64, "R": 64, "H": 2048, "N": 5632,
         "mixed": True, "rows": "requests"},
        # prompts of many requests in one batch
        {"name": "lora-prefill", "op": "lora", "T": 8191, "requests": 24, "G": 12, "R": 64, "H": 2048, "N": 2048,
         "mixed": True, "rows": "requests"},
        # one adapter on a down projection in training, ragged length
        {"name": "lora-grad-one", "op": "lora_grad", "T": 2047, "requests": 1, "G": 1, "R": 16, "H": 5632, "N": 2048,
         "mixed": False, "rows": "requests"},
        # an adapter per expert over rows that are sorted already
        {"name": "lora-grad-experts", "op": "lora_grad", "T": 16380, "requests": 60, "G": 60, "R": 32, "H": 2048,
         "N": 1408, "mixed": False, "rows": "experts"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["sort", "sort_grad", "combine_grad", "lora", "lora_grad"])
    if op in ("sort", "sort_grad", "combine_grad"):
        k = rng.randint(1, 8)
        E = rng.randint(max(8, k), 160)
        H = 8 * rng.randint(32, 400)
        most = 16383 * 6 * 2048 // (k * H)
        T = _log(rng, 1, min(32768, most))
        case = {"op": op, "T": T, "E": E, "k": k, "H": H}
        if op == "sort_grad":
            case["base"] = rng.random() < 0.5
        if op == "combine_grad":
            mode = rng.choice([ROUTE_QWEN, ROUTE_DEEPSEEK, ROUTE_SWITCH])
            case["mode"] = mode
            case["shared"] = mode != ROUTE_SWITCH and rng.random() < 0.7
            case["gate"] = case["shared"] and mode == ROUTE_QWEN
            case["capacity"] = case["seq"] = 0
            if mode == ROUTE_SWITCH:
                case["k"] = 1
                case["seq"] = seq = min(T, rng.choice([1, 37, 128, 512]))
                case["T"] = T // seq * seq
                case["capacity"] = max(1, 2 * seq // E)
        return case
    R = rng.choice([8, 16, 24, 32, 48, 64])
    H, N = 8 * rng.randint(32, 352), 8 * rng.randint(32, 704)
    if rng.random() < 0.5:
        H, N = N, H
    G = rng.randint(1, 24)
    most = 16380 * 32 * (2048 + 1408) // (R * (H + N))
    T = _log(rng, 1, min(8192, most))
    rows = rng.choice(["requests", "experts"])
    return {"op": op, "T": T, "requests": G if rows == "experts" else rng.randint(1, min(T, 64)), "G": G, "R": R,
            "H": H, "N": N, "mixed": rng.random() < 0.5, "rows": rows}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed, device):
    g = torch.Generator(device=device)
    g.manual_seed(int(seed) * 1000003 + 17)
    return g


def _normal(g, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def _route(case, seed):
    """k distinct experts a token, popular ones more often, and softmax weights."""
    T, E, k = case["T"], case["E"], case["k"]
    g = _gen(seed, "cuda")
    pop = torch.randperm(E, generator=g, device="cuda").float().add_(1.0).reciprocal_().log_()
    logits = pop + torch.randn(T, E, generator=g, device="cuda")
    w, idx = torch.softmax(logits, 1).topk(k, dim=1)
    return idx.to(torch.int32).contiguous(), w.contiguous(), g


def _requests(case, seed):
    """Rows of each group: adapter ids of the tokens, group offsets, and the
    tokens in the order of their adapters (those without one come last)."""
    T, G, n = case["T"], case["G"], min(case["T"], case["requests"])
    g = _gen(seed, "cpu")
    w = torch.rand(n, generator=g).add_(0.05)
    length = 1 + torch.floor(w / w.sum() * (T - n)).long()
    length[-1] += T - length.sum()
    if case["rows"] == "experts":
        ids = torch.repeat_interleave(torch.arange(n), length)
    else:
        # one request in twelve (never the first) uses no adapter
        who = torch.randint(0, G, (n,), generator=g)
        who[1:][torch.rand(n - 1, generator=g) < 1 / 12] = -1
        ids = torch.repeat_interleave(who, length)
    key = torch.where(ids < 0, G, ids)
    order = torch.argsort(key, stable=True)
    counts = torch.bincount(key, minlength=G + 1)[:G]
    offsets = torch.zeros(G + 1, dtype=torch.long)
    offsets[1:] = counts.cumsum(0)
    rank = torch.full((G,), case["R"])
    if case["mixed"]:
        rank = torch.randint(max(1, case["R"] // 4), case["R"] + 1, (G,), generator=g)
    i32 = torch.int32
    return {"ids": ids.to(i32).cuda(), "offsets": offsets.to(i32).cuda(), "rank": rank.to(i32).cuda(),
            "token_of_row": None if case["rows"] == "experts" else order.to(i32).cuda(), "most": int(counts.max())}


def prepare(case, seed):
    op = case["op"]
    s = dict(case)
    if op in ("lora", "lora_grad"):
        T, G, R, H, N = (case[n] for n in ("T", "G", "R", "H", "N"))
        s.update(_requests(case, seed))
        g = _gen(seed + 1, "cuda")
        keep = (torch.arange(R, device="cuda")[None, :] < s["rank"][:, None])
        # the adapters' share is about as large as the projection's own
        s["a"] = _normal(g, G, R, H, std=H ** -0.5) * keep[:, :, None]
        s["b"] = _normal(g, G, N, R, std=R ** -0.5) * keep[:, None, :]
        s["scale"] = torch.rand(G, generator=g, device="cuda") * 1.5 + 0.5
        s["x"] = _normal(g, T, H)
        if op == "lora":
            s["base"] = _normal(g, T, N)
        else:
            s["dy"] = _normal(g, T, N)
            s["base"] = _normal(g, T, H)
            # what the forward pass kept: x times the adapter's first matrix, by sorted row
            idx, ok = _padded(s)
            u = torch.bmm(s["x"][idx.reshape(-1)].view(G, -1, H).float(), s["a"].float().transpose(1, 2))
            s["u"] = torch.zeros(T, R, device="cuda")
            row = (s["offsets"][:-1, None] + torch.arange(idx.shape[1], device="cuda"))[ok]
            s["u"][row.long()] = u[ok]
        return s
    T, E, k, H = (case[n] for n in ("T", "E", "k", "H"))
    idx, w, g = _route(case, seed)
    if op == "sort":
        s["idx"], s["x"] = idx, _normal(g, T, H)
        return s
    if op == "combine_grad" and case["capacity"]:
        hot = torch.nn.functional.one_hot(idx[:, 0].long(), E).view(-1, case["seq"], E)
        late = (hot.cumsum(1) * hot).sum(2).reshape(T, 1) > case["capacity"]
        idx = torch.where(late, -1, idx).to(torch.int32)
    counts, offsets, row_of, token_of_row = _sorted(idx, E)
    rows = T * k                                           # as many as the layer's buffers hold
    s["row_of"], s["rows"] = row_of, rows
    if op == "sort_grad":
        s["dxp"] = _normal(g, rows, H, std=0.01)
        s["add"] = _normal(g, T, H, std=0.01) if case["base"] else None
        return s
    s["w"] = w
    s["dout"] = _normal(g, T, H, std=0.01)
    s["y"] = _normal(g, rows, H)
    s["dy"] = torch.zeros(rows, H, dtype=torch.bfloat16, device="cuda")   # rows behind the last expert's stay as they are
    s["ysh"] = _normal(g, T, H) if case["shared"] else None
    s["g"] = torch.rand(T, generator=g, device="cuda") if case["gate"] else None
    s["x"] = _normal(g, T, H) if case["mode"] == ROUTE_SWITCH else None
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _sorted(idx, E):
    """Rows of every (token, slot): grouped by expert, tokens ascending in each."""
    T, k = idx.shape
    hot = idx[:, :, None] == torch.arange(E, dtype=idx.dtype, device=idx.device)      # [T, k, E]
    upto = hot.any(1).to(torch.int32).cumsum(0, dtype=torch.int32)                     # tokens of e up to t
    counts = upto[-1]
    ends = counts.cumsum(0, dtype=torch.int32)
    offsets = torch.cat([torch.zeros_like(ends[:1]), ends])
    e = idx.clamp(min=0).long()
    row = offsets[e] + upto.gather(1, e) - 1
    row_of = torch.where(idx >= 0, row, -1).to(torch.int32)
    token_of_row = torch.empty(T * k + 1, dtype=torch.int32, device=idx.device)
    slot = torch.where(idx >= 0, row, T * k).long().reshape(-1)
    token_of_row[slot] = torch.arange(T, dtype=torch.int32, device=idx.device).repeat_interleave(k)
    return counts, offsets, row_of, token_of_row[:T * k]


def _padded(s):
    """Token of each (group, place), groups padded to the longest, and which places hold one."""
    place = s["offsets"][:-1, None] + torch.arange(s["most"], device="cuda")
    ok = place < s["offsets"][1:, None]
    row = torch.where(ok, place, 0).long()
    return (row if s["token_of_row"] is None else s["token_of_row"][row].long()), ok


def _add_rows(base, idx, ok, rows):
    """base plus each valid padded row at its token (a token has one row at most)."""
    out = torch.zeros(base.shape[0] + 1, base.shape[1], device="cuda")
    out[torch.where(ok, idx, base.shape[0])] = rows
    return (base.float() + out[:-1]).to(base.dtype)


def _plain(s):
    op = s["op"]
    if op == "sort":
        counts, offsets, row_of, token_of_row = _sorted(s["idx"], s["E"])
        return counts, offsets, row_of, token_of_row, s["x"][token_of_row.long()]
    if op == "sort_grad":
        kept = (s["row_of"] >= 0)[:, :, None]
        dx = (s["dxp"][s["row_of"].clamp(min=0).long()].float() * kept).sum(1)
        return (dx if s["add"] is None else dx + s["add"].float()).to(torch.bfloat16)
    if op == "combine_grad":
        r, dout = s["row_of"].clamp(min=0).long(), s["dout"].float()
        kept = s["row_of"] >= 0
        w = s["w"]
        dy = torch.zeros(s["rows"] + 1, s["H"], dtype=torch.bfloat16, device="cuda")
        dy[torch.where(kept, r, s["rows"])] = (w[:, :, None] * dout[:, None]).to(torch.bfloat16)
        dw = (s["y"][r].float() * dout[:, None]).sum(2)
        passed = 0.0 if s["x"] is None else (s["x"].float() * dout).sum(1, keepdim=True)
        out = {"dy": dy[:-1], "dw": torch.where(kept, dw, passed)}
        if s["ysh"] is not None:
            out["dysh"] = (dout if s["g"] is None else s["g"][:, None] * dout).to(torch.bfloat16)
        if s["g"] is not None:
            out["dg"] = (dout * s["ysh"].float()).sum(1)
        if s["mode"] == ROUTE_SWITCH:
            out["dx"] = torch.where(kept, 0.0, w * dout).to(torch.bfloat16)
        return out
    idx, ok = _padded(s)
    a, b, scale = s["a"].float(), s["b"].float(), s["scale"][:, None, None]
    x = s["x"][idx].float() * ok[:, :, None]
    if op == "lora":
        return _add_rows(s["base"], idx, ok, torch.bmm(torch.bmm(x, a.transpose(1, 2)) * scale, b.transpose(1, 2)))
    dy = s["dy"][idx].float() * ok[:, :, None] * scale
    row = torch.where(ok, s["offsets"][:-1, None] + torch.arange(s["most"], device="cuda"), 0)
    u = s["u"][row.long()] * ok[:, :, None]
    v = torch.bmm(dy, b)
    return {"dx": _add_rows(s["base"], idx, ok, torch.bmm(v, a)),
            "da": torch.bmm(v.transpose(1, 2), x).to(s["a"].dtype),
            "db": torch.bmm(dy.transpose(1, 2), u).to(s["b"].dtype)}


def run(state):
    s = state
    if not own:
        return _plain(s)
    ops = _ops()
    op = s["op"]
    if op == "sort":
        return ops.permute(s["idx"], s["x"], s["E"])
    if op == "sort_grad":
        return ops.permute_grad(s["dxp"], s["row_of"], base=s["add"])
    if op == "combine_grad":
        got = ops.combine_grad(s["dout"], s["y"], s["row_of"], s["w"], s["mode"], y_shared=s["ysh"],
                               shared_gate=s["g"], x=s["x"], dy=s["dy"])
        return {n: t for n, t in zip(("dy", "dw", "dysh", "dg", "dx"), got) if t is not None}
    if op == "lora":
        return ops.lora(s["x"], s["base"], s["a"], s["b"], s["scale"], s["offsets"],
                        token_of_row=s["token_of_row"], rank=s["rank"])
    dx, da, db = ops.lora_grad(s["dy"], s["x"], s["u"], s["a"], s["b"], s["scale"], s["offsets"],
                               token_of_row=s["token_of_row"], rank=s["rank"], base=s["base"])
    return {"dx": dx, "da": da, "db": db}


def work(case):
    op = case["op"]
    if op in ("lora", "lora_grad"):
        T, R, H, N = (case[n] for n in ("T", "R", "H", "N"))
        G = min(case["G"], case["requests"], T)
        if case["mixed"]:
            R = (max(1, R // 4) + R) / 2                   # the ranks' mean
        if op == "lora":
            return {"bytes": 2 * T * (H + 2 * N) + 2 * G * R * (H + N) + 4 * T, "flops": 2 * T * R * (H + N)}
        return {"bytes": 2 * T * (3 * H + N) + 4 * T * R + 4 * G * R * (H + N) + 4 * T, "flops": 4 * T * R * (H + N)}
    T, k, H = case["T"], case["k"], case["H"]
    row = 2 * T * H
    if op == "sort":
        return {"bytes": row * (1 + k) + 12 * T * k, "flops": 0}
    if op == "sort_grad":
        return {"bytes": row * (k + 1 + int(case["base"])) + 4 * T * k, "flops": T * k * H}
    more = (2 if case["shared"] else 0) - (0 if case["gate"] or not case["shared"] else 1)
    more += 1 if case["mode"] == ROUTE_SWITCH else 0
    return {"bytes": row * (1 + 2 * k + more) + 12 * T * k, "flops": 3 * T * k * H}


# ---------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "sort":
        per = [torch.nonzero((s["idx"] == e).any(1))[:, 0] for e in range(case["E"])]
        return None, None, None, None, s["x"].double()[torch.cat(per)]
    if op == "sort_grad":
        k, T = case["k"], case["T"]
        at = s["row_of"].reshape(-1).long()
        tok = torch.arange(T, device="cuda").repeat_interleave(k)
        dx = torch.zeros(T, case["H"], dtype=torch.float64, device="cuda") if s["add"] is None else s["add"].double()
        return dx.index_add(0, tok[at >= 0], s["dxp"].double()[at[at >= 0]])
    if op == "combine_grad":
        T, k, dout = case["T"], case["k"], s["dout"].double()
        w = s["w"].double()
        dy = torch.zeros(s["rows"], case["H"], dtype=torch.float64, device="cuda")
        dw = torch.zeros(T, k, dtype=torch.float64, device="cuda")
        for j in range(k):
            t = torch.nonzero(s["row_of"][:, j] >= 0)[:, 0]
            r = s["row_of"][t, j].long()
            dy[r] = w[t, j, None] * dout[t]
            dw[t, j] = torch.einsum("th,th->t", s["y"][r].double(), dout[t])
        out = {"dy": dy, "dw": dw}
        if case["mode"] == ROUTE_SWITCH:
            gone = torch.nonzero(s["row_of"][:, 0] < 0)[:, 0]
            dx = torch.zeros(T, case["H"], dtype=torch.float64, device="cuda")
            dx[gone] = w[gone] * dout[gone]
            dw[gone, 0] = torch.einsum("th,th->t", s["x"][gone].double(), dout[gone])
            out["dx"] = dx
        if case["shared"]:
            out["dysh"] = dout if s["g"] is None else torch.einsum("t,th->th", s["g"].double(), dout)
        if case["gate"]:
            out["dg"] = torch.einsum("th,th->t", dout, s["ysh"].double())
        return out
    off = s["offsets"].tolist()
    out = s["base"].double()
    da, db = torch.zeros_like(s["a"], dtype=torch.float64), torch.zeros_like(s["b"], dtype=torch.float64)
    for g in range(case["G"]):
        if off[g + 1] == off[g]:
            continue
        rows = torch.arange(off[g], off[g + 1], device="cuda")
        t = rows if s["token_of_row"] is None else s["token_of_row"][rows].long()
        A, B, c = s["a"][g].double(), s["b"][g].double(), float(s["scale"][g])
        if op == "lora":
            out[t] += c * (s["x"][t].double() @ A.T @ B.T)
        else:
            dy = s["dy"][t].double()
            v = c * (dy @ B)
            out[t] += v @ A
            da[g] = v.T @ s["x"][t].double()
            db[g] = c * (dy.T @ s["u"][rows].double())
    return out if op == "lora" else {"dx": out, "da": da, "db": db}
