"""The expert-layer operators and what is measured of them: routing (the
pattern of a top-k routing matrix, its weighted combine and the combine's
gradient), products grouped by expert over ragged row ranges, and the dense
product with bias, activation and residual in its epilogue.

`run` computes a case either in plain torch operations (own = False) or
through the framework's operators (own = True).  Sizes are generic.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f32": 4}


# ------------------------------------------------------------------ cases

def listed():
    return [
        # routing: the pattern for a decode step of a few dozen sequences
        {"name": "route_decode", "op": "route", "T": 37, "k": 4, "E": 64, "drop": 0.0},
        # routing: the pattern for a whole batch of prompts, with dropped entries
        {"name": "route_prefill", "op": "route", "T": 60001, "k": 8, "E": 256, "drop": 0.02},
        # the experts' rows summed back into their tokens after a prefill chunk
        {"name": "combine", "op": "combine", "T": 8191, "k": 4, "E": 64, "N": 4096, "dt": "bf16",
         "drop": 0.02},
        # gradient of the combine in a training step
        {"name": "combine_bwd", "op": "combine_bwd", "T": 4096, "k": 8, "E": 64, "N": 2048,
         "dt": "bf16", "drop": 0.0},
        # one decode step of a layer of experts: a row or two per expert
        {"name": "grouped_decode", "op": "grouped", "T": 24, "k": 2, "E": 32, "K": 2048, "N": 4096,
         "dt": "bf16", "act": "silu", "order": "row", "skew": 0.5, "drop": 0.0},
        # a prefill chunk through the experts' first product, skewed row counts
        {"name": "grouped_prefill", "op": "grouped", "T": 8011, "k": 4, "E": 32, "K": 2048,
         "N": 4096, "dt": "bf16", "act": "silu", "order": "row", "skew": 0.7, "drop": 0.0},
        # the experts' gradients in a training step
        {"name": "grouped_bwd", "op": "grouped_bwd", "T": 4096, "k": 2, "E": 16, "K": 2048,
         "N": 4096, "dt": "bf16", "act": "silu", "order": "row", "skew": 0.5, "drop": 0.01},
        # the grouped product in single precision, an odd width
        {"name": "grouped_f32", "op": "grouped", "T": 701, "k": 2, "E": 8, "K": 1024, "N": 1001,
         "dt": "f32", "act": "none", "order": "col", "skew": 0.5, "drop": 0.0},
        # one token through a dense layer
        {"name": "fused_token", "op": "fused", "M": 1, "K": 4096, "N": 4096, "dt": "bf16",
         "act": "gelu", "order": "row", "residual": False, "keep": False},
        # a training batch through a wide dense layer, the pre-activation kept
        {"name": "fused_train", "op": "fused", "M": 8192, "K": 4096, "N": 16384, "dt": "bf16",
         "act": "gelu", "order": "row", "residual": False, "keep": True},
        # its gradients, an odd number of rows
        {"name": "fused_bwd", "op": "fused_bwd", "M": 4099, "K": 2048, "N": 8192, "dt": "bf16",
         "act": "gelu", "order": "row"},
        # odd sizes with a residual, as a small projection has them
        {"name": "fused_odd", "op": "fused", "M": 333, "K": 1023, "N": 2049, "dt": "bf16",
         "act": "none", "order": "col", "residual": True, "keep": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A layer width: mostly multiples of 128, some of 8, some odd."""
    step = rng.choice([128, 128, 128, 8, 1])
    n = _log(rng, lo, hi)
    n = n | 1 if step == 1 else max(step, n // step * step)
    return n + step if n == 3 * 1024 else n


def draw(rng):
    op = rng.choice(["route", "combine", "combine_bwd", "grouped", "grouped", "grouped_bwd",
                     "fused", "fused", "fused_bwd"])
    dt = rng.choice(["bf16", "bf16", "bf16", "f32"])
    drop = rng.choice([0.0, 0.0, 0.02])
    order = rng.choice(["row", "row", "col"])
    act = rng.choice(["none", "relu", "silu", "gelu"])
    if op == "route":
        E = _log(rng, 4, 256)
        return {"op": op, "T": _log(rng, 1, 60000), "k": min(rng.randint(1, 8), E), "E": E,
                "drop": drop}
    if op in ("combine", "combine_bwd"):
        k, N = rng.randint(1, 8), _width(rng, 256, 8192)
        T = _log(rng, 1, max(1, (1 << 27) // (k * N)))
        return {"op": op, "T": T, "k": k, "E": 64, "N": N, "dt": dt, "drop": drop}
    big = 4.0e11 if dt == "bf16" else 6.0e10            # flops of one pass, at most
    if op in ("grouped", "grouped_bwd"):
        E = _log(rng, 4, 128)
        K, N = _width(rng, 256, 4096), _width(rng, 256, 4096)
        while E * K * N > 1 << 29:
            E = max(4, E // 2)
        k = min(rng.randint(1, 4), E)
        lo = 1 if op == "grouped" else 64
        most = big / ((2 if op == "grouped" else 4) * k * K * N)
        T = _log(rng, lo, max(lo, int(min(16384, most))))
        return {"op": op, "T": T, "k": k, "E": E, "K": K, "N": N, "dt": dt, "act": act,
                "order": order, "skew": rng.choice([0.0, 0.5, 1.0]), "drop": drop}
    K, N = _width(rng, 256, 8192), _width(rng, 256, 8192)
    lo = 1 if op == "fused" else 64
    M = _log(rng, lo, max(lo, int(min(16384, big / ((2 if op == "fused" else 4) * K * N)))))
    case = {"op": op, "M": M, "K": K, "N": N, "dt": dt, "act": act, "order": order}
    if op == "fused":
        case |= {"residual": rng.random() < 0.5, "keep": act != "none" and rng.random() < 0.3}
    return case


# ----------------------------------------------------------------- inputs

def _ids(T, k, E, skew, drop, g):
    """k distinct experts a token, their popularity spread by `skew`; a
    dropped entry (capacity reached, padding) is -1."""
    logits = skew * torch.randn(E, generator=g, device="cuda")
    u = torch.rand(T, E, generator=g, device="cuda").clamp_min_(1e-9)
    ids = (logits - torch.log(-torch.log(u))).topk(k, dim=1).indices.to(torch.int32)
    if drop:
        ids = torch.where(torch.rand(T, k, generator=g, device="cuda") < drop,
                          torch.full_like(ids, -1), ids)
    return ids.contiguous()


def _pattern(ids, E):
    """rowptr, source, slot of the routing pattern, in torch operations."""
    T, k = ids.shape
    flat = ids.reshape(-1).to(torch.int64)
    key = torch.where((flat < 0) | (flat >= E), torch.full_like(flat, E), flat)
    order = torch.sort(key, stable=True).indices
    counts = (key[:, None] == torch.arange(E, device=key.device)).sum(0)
    rowptr = torch.zeros(E + 1, dtype=torch.int64, device=key.device)
    rowptr[1:] = counts.cumsum(0)
    place = torch.empty_like(order)
    place[order] = torch.arange(T * k, device=key.device)
    slot = torch.where(key == E, torch.full_like(place, -1), place)
    live = torch.arange(T * k, device=key.device) < rowptr[E]
    source = torch.where(live, order // k, torch.full_like(order, -1))
    return (rowptr.to(torch.int32), source.to(torch.int32), slot.reshape(T, k).to(torch.int32))


def _normal(shape, dt, g, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(_DT[dt])


def _weight(E, K, N, dt, order, g):
    """E matrices K x N, stored row-major or (order "col") as N x K."""
    shape = (E, K, N) if order == "row" else (E, N, K)
    w = torch.empty(shape, dtype=_DT[dt], device="cuda")
    for e in range(E):
        w[e] = _normal(shape[1:], dt, g, K ** -0.5)
    return w if order == "row" else w.transpose(1, 2)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s, op, dt = dict(case), case["op"], case.get("dt", "bf16")
    if own:
        import jlust_b200
        s["J"] = jlust_b200
    if op == "route":
        s["ids"] = _ids(case["T"], case["k"], case["E"], 0.5, case["drop"], g)
        return s
    if op in ("combine", "combine_bwd"):
        T, k, N = case["T"], case["k"], case["N"]
        s["pattern"] = _pattern(_ids(T, k, case["E"], 0.5, case["drop"], g), case["E"])
        s["g"] = torch.softmax(torch.randn(T, k, generator=g, device="cuda"), 1)
        s["z"] = _normal((T * k, N), dt, g)
        if op == "combine_bwd":
            s["dy"] = _normal((T, N), dt, g)
        if own:
            s["routing"] = s["J"].Routing(*s["pattern"])
        return s
    K, N, act = case["K"], case["N"], case["act"]
    if op in ("grouped", "grouped_bwd"):
        T, k, E = case["T"], case["k"], case["E"]
        rowptr, source, _ = _pattern(_ids(T, k, E, case["skew"], case["drop"], g), E)
        s["rowptr"], s["rows"] = rowptr, source
        s["at"] = rowptr.tolist()           # a plain program loops over the experts on the host
        s["x"] = _normal((T, K), dt, g)
        s["w"] = _weight(E, K, N, dt, case["order"], g)
        s["b"] = _normal((E, N), dt, g, 0.1)
        if op == "grouped_bwd":
            s["dy"] = _normal((T * k, N), dt, g)
            s["z"] = _normal((T * k, N), dt, g) if act != "none" else None
        elif own:
            s["handle"] = s["J"].prepare(s["J"].B200Backend(), s["J"].GroupedMMOp, s["w"],
                                         bias=s["b"], act=act)
        return s
    M = case["M"]
    s["x"] = _normal((M, K), dt, g)
    s["w"] = _weight(1, K, N, dt, case["order"], g)[0]
    s["b"] = _normal((N,), dt, g, 0.1)
    if op == "fused_bwd":
        s["dy"] = _normal((M, N), dt, g)
        s["z"] = _normal((M, N), dt, g) if act != "none" else None
        return s
    s["r"] = _normal((M, N), dt, g) if case["residual"] else None
    if own and not case["keep"]:
        s["handle"] = s["J"].prepare(s["J"].B200Backend(), s["J"].FusedMMOp, s["w"], bias=s["b"],
                                     act=act)
    return s


# ------------------------------------------------------------- plain forms

def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * (0.5 ** 0.5)))
    return z


def _dact(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return (0.5 * (1 + torch.erf(z * (0.5 ** 0.5)))
                + z * torch.exp(-0.5 * z * z) * ((2 * math.pi) ** -0.5))
    return torch.ones_like(z)


def _plain_combine(s):
    slot, dt = s["pattern"][2].to(torch.int64), _DT[s["dt"]]
    y = 0
    for j in range(s["k"]):
        live = slot[:, j] >= 0
        g = torch.where(live, s["g"][:, j], torch.zeros_like(s["g"][:, j]))
        y = y + g[:, None] * s["z"][slot[:, j].clamp_min(0)].float()
    return y.to(dt)


def _plain_combine_bwd(s):
    slot, dt = s["pattern"][2].to(torch.int64), _DT[s["dt"]]
    dy = s["dy"].float()
    dz = torch.zeros_like(s["z"])
    dg = []
    for j in range(s["k"]):
        live = slot[:, j] >= 0
        rows = s["z"][slot[:, j].clamp_min(0)].float()
        dg.append(torch.where(live, (rows * dy).sum(1), torch.zeros_like(dy[:, 0])))
        at = slot[:, j][live]
        dz[at] = (s["g"][:, j][:, None] * dy)[live].to(dt)
    return {"dz": dz, "dg": torch.stack(dg, 1)}


def _plain_grouped(s):
    dt = _DT[s["dt"]]
    y = torch.zeros(s["T"] * s["k"], s["N"], dtype=dt, device="cuda")
    for e in range(s["E"]):
        a, b = s["at"][e], s["at"][e + 1]
        if b > a:
            z = s["x"][s["rows"][a:b].to(torch.int64)].float() @ s["w"][e].float()
            y[a:b] = _act(z + s["b"][e].float(), s["act"]).to(dt)
    return y


def _plain_grouped_bwd(s):
    dt = _DT[s["dt"]]
    dx = torch.zeros(s["T"] * s["k"], s["K"], dtype=dt, device="cuda")
    dw = torch.zeros(s["E"], s["K"], s["N"], dtype=dt, device="cuda")
    db = torch.zeros(s["E"], s["N"], dtype=dt, device="cuda")
    for e in range(s["E"]):
        a, b = s["at"][e], s["at"][e + 1]
        if b > a:
            dz = s["dy"][a:b].float()
            if s["z"] is not None:
                dz = dz * _dact(s["z"][a:b].float(), s["act"])
            dx[a:b] = (dz @ s["w"][e].float().t()).to(dt)
            dw[e] = (s["x"][s["rows"][a:b].to(torch.int64)].float().t() @ dz).to(dt)
            db[e] = dz.sum(0).to(dt)
    return {"dx": dx, "dw": dw, "db": db}


def _plain_fused(s):
    z = s["x"].float() @ s["w"].float() + s["b"].float()
    y = _act(z, s["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    dt = _DT[s["dt"]]
    return {"y": y.to(dt), "z": z.to(dt)} if s["keep"] else y.to(dt)


def _plain_fused_bwd(s):
    dt = _DT[s["dt"]]
    dz = s["dy"].float()
    if s["z"] is not None:
        dz = dz * _dact(s["z"].float(), s["act"])
    return {"dx": (dz @ s["w"].float().t()).to(dt), "dw": (s["x"].float().t() @ dz).to(dt),
            "db": dz.sum(0).to(dt)}


_PLAIN = {"route": lambda s: dict(zip(("rowptr", "source", "slot"), _pattern(s["ids"], s["E"]))),
          "combine": _plain_combine, "combine_bwd": _plain_combine_bwd,
          "grouped": _plain_grouped, "grouped_bwd": _plain_grouped_bwd,
          "fused": _plain_fused, "fused_bwd": _plain_fused_bwd}


# --------------------------------------------------- the framework's calls

def _own(s):
    J, op = s["J"], s["op"]
    if op == "route":
        r = J.route(s["ids"], s["E"])
        return {"rowptr": r.rowptr, "source": r.source, "slot": r.slot}
    if op == "combine":
        return J.combine(s["z"], s["routing"], s["g"])
    if op == "combine_bwd":
        dz, dg = J.combine_backward(s["dy"], s["z"], s["routing"], s["g"])
        return {"dz": dz, "dg": dg}
    if op == "grouped":
        return J.execute(s["handle"], s["x"], s["rowptr"], rows=s["rows"])
    if op == "grouped_bwd":
        dx, dw, db = J.grouped_matmul_backward(s["dy"], s["x"], s["w"], s["rowptr"],
                                               rows=s["rows"], z=s["z"], act=s["act"], bias=True)
        return {"dx": dx, "dw": dw, "db": db}
    if op == "fused_bwd":
        dx, dw, db = J.fused_matmul_backward(s["dy"], s["x"], s["w"], z=s["z"], act=s["act"],
                                             bias=True)
        return {"dx": dx, "dw": dw, "db": db}
    if s["keep"]:
        y, z = J.fused_matmul(s["x"], s["w"], bias=s["b"], act=s["act"], residual=s["r"],
                              keep_preact=True)
        return {"y": y, "z": z}
    return J.execute(s["handle"], s["x"], residual=s["r"])


def run(state):
    return _own(state) if own else _PLAIN[state["op"]](state)


# -------------------------------------------------------------- accounting

def work(case):
    op = case["op"]
    if op == "route":
        n = case["T"] * case["k"]
        return {"bytes": 12 * n + 4 * (case["E"] + 1), "flops": 0}
    b = _SIZE[case["dt"]]
    if op in ("combine", "combine_bwd"):
        S, T, N = case["T"] * case["k"], case["T"], case["N"]
        live = 1 - case["drop"]
        if op == "combine":
            return {"bytes": (live * S + T) * N * b + 8 * S, "flops": 2 * live * S * N}
        return {"bytes": (live * S + S + T) * N * b + 12 * S, "flops": 3 * live * S * N}
    K, N = case["K"], case["N"]
    kept = case["act"] != "none"
    if op in ("grouped", "grouped_bwd"):
        T, S, E = case["T"], case["T"] * case["k"], case["E"]
        live = S * (1 - case["drop"])
        # experts that any row reaches, for rows spread evenly
        used = E * (1 - (1 - 1 / E) ** live)
        if op == "grouped":
            return {"bytes": (T * K + used * (K * N + N) + S * N) * b + 4 * S + 4 * (E + 1),
                    "flops": 2 * live * K * N}
        return {"bytes": ((1 + kept) * live * N + T * K + used * K * N + S * K + E * (K * N + N)) * b
                + 4 * S + 4 * (E + 1), "flops": 4 * live * K * N}
    M = case["M"]
    if op == "fused":
        outs = 1 + bool(case["residual"]) + bool(case["keep"])
        return {"bytes": (M * K + K * N + N + outs * M * N) * b, "flops": 2 * M * K * N}
    return {"bytes": ((1 + kept) * M * N + 2 * M * K + 2 * K * N + N) * b, "flops": 4 * M * K * N}


# ------------------------------------------- the definitions, in 64 bits

def _act64(z, act):
    if act == "silu":
        return z * torch.special.expit(z)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    return z.clamp_min(0) if act == "relu" else z


def _dact64(z, act):
    if act == "silu":
        p = torch.special.expit(z)
        return p + z * p * torch.special.expit(-z)
    if act == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)
    return torch.heaviside(z, torch.zeros_like(z)) if act == "relu" else torch.ones_like(z)


def exact(case, seed):
    s = prepare(case, seed)
    op, dbl = case["op"], torch.float64
    if op == "route":
        return None                      # whole numbers: compared as they are
    if op in ("combine", "combine_bwd"):
        T, N, S = case["T"], case["N"], case["T"] * case["k"]
        slot = s["pattern"][2].to(torch.int64)
        t, j = torch.nonzero(slot >= 0, as_tuple=True)
        p, gate = slot[t, j], s["g"][t, j].to(dbl)
        step = max(1, (1 << 26) // N)    # entries at a time
        if op == "combine":
            y = torch.zeros(T, N, dtype=dbl, device="cuda")
            for i in range(0, t.numel(), step):
                c = slice(i, i + step)
                y.index_add_(0, t[c], gate[c, None] * s["z"][p[c]].to(dbl))
            return y
        dz = torch.zeros(S, N, dtype=dbl, device="cuda")
        dg = torch.zeros(T, case["k"], dtype=dbl, device="cuda")
        for i in range(0, t.numel(), step):
            c = slice(i, i + step)
            dy = s["dy"][t[c]].to(dbl)
            dz[p[c]] = gate[c, None] * dy
            dg[t[c], j[c]] = torch.linalg.vecdot(dy, s["z"][p[c]].to(dbl))
        return {"dz": dz, "dg": dg}
    act = case["act"]
    if op == "fused":
        z = torch.addmm(s["b"].to(dbl), s["x"].to(dbl), s["w"].to(dbl))
        y = _act64(z, act)
        if s["r"] is not None:
            y += s["r"].to(dbl)
        return {"y": y, "z": z} if case["keep"] else y
    if op == "fused_bwd":
        dz = s["dy"].to(dbl)
        if s["z"] is not None:
            dz = dz * _dact64(s["z"].to(dbl), act)
        return {"dx": torch.mm(dz, s["w"].to(dbl).T), "dw": torch.mm(s["x"].to(dbl).T, dz),
                "db": dz.sum(0)}
    # grouped: each expert's rows by the expert of each slot
    E, K, N, S = case["E"], case["K"], case["N"], case["T"] * case["k"]
    ends = s["rowptr"][1:].to(torch.int64)
    expert = torch.searchsorted(ends, torch.arange(S, device="cuda"), right=True)
    if op == "grouped":
        y = torch.zeros(S, N, dtype=dbl, device="cuda")
    else:
        dx = torch.zeros(S, K, dtype=dbl, device="cuda")
        dw = torch.zeros(E, K, N, dtype=dbl, device="cuda")
        db = torch.zeros(E, N, dtype=dbl, device="cuda")
    for e in range(E):
        p = torch.nonzero(expert == e)[:, 0]
        if not p.numel():
            continue
        x, w = s["x"][s["rows"][p].to(torch.int64)].to(dbl), s["w"][e].to(dbl)
        if op == "grouped":
            y[p] = _act64(torch.addmm(s["b"][e].to(dbl), x, w), act)
        else:
            dz = s["dy"][p].to(dbl)
            if s["z"] is not None:
                dz = dz * _dact64(s["z"][p].to(dbl), act)
            dx[p], dw[e], db[e] = torch.mm(dz, w.T), torch.mm(x.T, dz), dz.sum(0)
    return y if op == "grouped" else {"dx": dx, "dw": dw, "db": db}
