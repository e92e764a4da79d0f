"""A layer of experts on the framework's operators: one training step and one
decode step, each checked against plain torch.

    python examples/expert_layer.py [--tokens 4096] [--experts 16] [--top-k 2]
                                    [--width 1024] [--hidden 2048] [--steps 20]

The layer: a dense projection with residual (fused_matmul), top-k routing
(route), the experts' two products over ragged groups (grouped_matmul) and the
weighted sum of a token's rows (combine); then every gradient.  Needs a B200.
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import jlust_b200 as J  # noqa: E402


def make(a, dtype=torch.bfloat16, device="cuda"):
    g = torch.Generator(device=device).manual_seed(a.seed)

    def t(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=device) * scale).to(dtype)

    D, H, E = a.width, a.hidden, a.experts
    return {"wp": t(D, D, scale=D ** -0.5), "bp": t(D, scale=0.1), "wr": t(D, E, scale=D ** -0.5),
            "w1": t(E, D, H, scale=D ** -0.5), "b1": t(E, H, scale=0.1),
            "w2": t(E, H, D, scale=H ** -0.5)}, t


def choose(p, h, k):
    """Each token's k experts and their weights (plain torch: the router's
    scores are a small dense product)."""
    scores, ids = (h @ p["wr"]).float().topk(k, dim=1)
    return ids.to(torch.int32), torch.softmax(scores, 1)


def forward(p, x, k):
    """The layer's output and what its gradients need."""
    h, zp = J.fused_matmul(x, p["wp"], bias=p["bp"], act="gelu", residual=x, keep_preact=True)
    ids, gates = choose(p, h, k)
    r = J.route(ids, p["w1"].shape[0])
    a, z = J.grouped_matmul(h, p["w1"], r.rowptr, rows=r.source, bias=p["b1"], act="silu",
                            keep_preact=True)
    o = J.grouped_matmul(a, p["w2"], r.rowptr)
    return J.combine(o, r, gates), (h, zp, r, gates, a, z, o)


def backward(p, x, saved, dy):
    """Gradients of the layer (the choice of experts and the gates' own path
    into the router left to the caller, who has d gates)."""
    h, zp, r, gates, a, z, o = saved
    do, dgates = J.combine_backward(dy, o, r, gates)
    da, dw2, _ = J.grouped_matmul_backward(do, a, p["w2"], r.rowptr)
    dhs, dw1, db1 = J.grouped_matmul_backward(da, h, p["w1"], r.rowptr, rows=r.source, z=z,
                                              act="silu", bias=True)
    dh = J.combine(dhs, r)                      # a token's rows summed
    dx, dwp, dbp = J.fused_matmul_backward(dh, x, p["wp"], z=zp, act="gelu", bias=True)
    return {"x": dx + dh, "wp": dwp, "bp": dbp, "w1": dw1, "b1": db1, "w2": dw2, "gates": dgates}


def plain(p, x, ids, gates, dy):
    """The same in torch, fp32 with autograd, expert by expert."""
    q = {n: t.float().requires_grad_() for n, t in p.items()}
    xf, gf = x.float().requires_grad_(), gates.detach().clone().requires_grad_()
    h = torch.nn.functional.gelu(xf @ q["wp"] + q["bp"]) + xf
    y = torch.zeros_like(h)
    for e in range(p["w1"].shape[0]):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        if t.numel():
            o = torch.nn.functional.silu(h[t] @ q["w1"][e] + q["b1"][e]) @ q["w2"][e]
            y = y.index_add(0, t, gf[t, j, None] * o)
    y.backward(dy.float())
    return y.detach(), {"x": xf.grad, "wp": q["wp"].grad, "bp": q["bp"].grad, "w1": q["w1"].grad,
                        "b1": q["b1"].grad, "w2": q["w2"].grad, "gates": gf.grad}


def relative(a, b):
    return ((a.float() - b).norm() / b.norm().clamp_min(1e-30)).item()


def main(argv=None):
    ap = argparse.ArgumentParser()
    for name, value in (("tokens", 4096), ("experts", 16), ("top-k", 2), ("width", 1024),
                        ("hidden", 2048), ("steps", 20), ("seed", 0)):
        ap.add_argument(f"--{name}", type=int, default=value)
    a = ap.parse_args(argv)
    p, t = make(a)
    x, dy = t(a.tokens, a.width), t(a.tokens, a.width)

    y, saved = forward(p, x, a.top_k)
    grads = backward(p, x, saved, dy)
    J.device_status()
    r, gates = saved[2], saved[3]
    ids = torch.full_like(r.slot, -1)           # the experts back from the pattern
    expert = torch.searchsorted(r.rowptr[1:], torch.arange(r.n_slots, device=x.device), right=True)
    ids[:] = expert[r.slot.long()].to(torch.int32)
    ry, rgrads = plain(p, x, ids, gates, dy)
    worst = max([relative(y, ry)] + [relative(grads[n], rgrads[n]) for n in grads])
    print(f"training step: largest relative difference from fp32 torch {worst:.2e}")
    assert worst < 2e-2                         # bf16 activations through three products

    one = t(1, a.width)                         # decode: one token, prepared products
    be = J.B200Backend()
    hp = J.prepare(be, J.FusedMMOp, p["wp"], bias=p["bp"], act="gelu")
    h1 = J.prepare(be, J.GroupedMMOp, p["w1"], bias=p["b1"], act="silu")
    h2 = J.prepare(be, J.GroupedMMOp, p["w2"])

    def decode(x):
        h = J.execute(hp, x, residual=x)
        ids, gates = choose(p, h, a.top_k)
        r = J.route(ids, a.experts)
        return J.combine(J.execute(h2, J.execute(h1, h, r.rowptr, rows=r.source), r.rowptr), r, gates)

    assert relative(decode(one), forward(p, one, a.top_k)[0].float()) < 1e-2

    def timed(f):
        f()
        torch.cuda.synchronize()
        at = time.perf_counter()
        for _ in range(a.steps):
            f()
        torch.cuda.synchronize()
        return (time.perf_counter() - at) / a.steps * 1e6

    def step():
        _, s = forward(p, x, a.top_k)
        backward(p, x, s, dy)

    print(f"training step {timed(step):.0f} us ({a.tokens} tokens), decode {timed(lambda: decode(one)):.0f} us")


if __name__ == "__main__":
    main()
