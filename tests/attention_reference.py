"""node_attention restated in float64 torch operations, with its gradients and
elementwise bounds on what a float32-accumulating kernel may differ by
(test_node_attention.py).

Bounds, with u = 2^-24, h = half a step of the element type (0 for float32,
whose operands enter the products exactly) and n the longest sum:
  dw: error of a score in nats.  A product sum of C terms is off by at most (C +
      1) u sum|q||k|; scaling, tanh, the bias and the change to log 2 units and
      back add at most 8 roundings of the largest magnitude in play, and the
      final subtraction of the statistics 4 more.
  p:  relative error 2 dw (numerator and normaliser) + (n + 8) u.
  o:  sum p |dv| <= max over v of (p's error + 2 h: p is rounded to the type, the
      normaliser is not; and the result is rounded) + (n + 8) u.
  t = p (gp - D) slack: p's error on |gp - D|, the products' errors (C + 1) u
      sum|go||v| in gp, D's error |go| (error of o), slack's error (2 |z/cap|
      times tanh's 8 u), and h for its own rounding."""
import math

import torch

U = 2.0 ** -24
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def per_graph(q, k, v, q_ptr, k_ptr):
    for b in range(len(q_ptr) - 1):
        yield b, slice(q_ptr[b], q_ptr[b + 1]), slice(k_ptr[b], k_ptr[b + 1])


def reference(q, k, v, q_ptr, k_ptr, dist=None, slope=None, scale=None, cap=0.0, grad=None):
    """dict of out, and with grad also q, k, v, slope, each a (value, bound) pair
    in float64.  q_ptr, k_ptr: python lists."""
    dt = q.dtype
    h, step = HALF[dt], (HALF[dt] or U)
    # a half type's values below its smallest normal step round by up to half that step
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}.get(dt, 2.0 ** -150)
    H, Hk, C = q.shape[1], k.shape[1], q.shape[2]
    G = H // Hk
    scale = 1.0 / math.sqrt(C) if scale is None else scale
    q, k, v = q.detach().double(), k.detach().double(), v.detach().double()
    z8 = lambda t: torch.zeros_like(t)  # noqa: E731
    out, out_b, gq, gq_b = z8(q), z8(q), z8(q), z8(q)
    gk, gk_b, gv, gv_b = z8(k), z8(k), z8(k), z8(k)
    gs = torch.zeros(H, dtype=torch.float64, device=q.device)
    gs_b = gs.clone()
    for b, rq, rk in per_graph(q, k, v, q_ptr, k_ptr):
        nq, nk = rq.stop - rq.start, rk.stop - rk.start
        if nq <= 0 or nk <= 0:
            continue
        n = max(nq * G, nk)
        d = torch.zeros(nq, nk, dtype=torch.float64, device=q.device)
        if dist is not None:
            d.fill_(math.inf)
            m = (dist if dist.dim() == 2 else dist[b])[:nq, :nk].double()
            d[:m.shape[0], :m.shape[1]] = m
        seen = torch.isfinite(d)
        d = torch.where(seen, d, 0.0)
        for head in range(H):
            qq, kk, vv = q[rq, head], k[rk, head // G], v[rk, head // G]
            s = 0.0 if slope is None else float(slope[head])
            raw = (qq @ kk.T) * scale
            z = cap * torch.tanh(raw / cap) if cap else raw
            w = torch.where(seen, z - s * d, -math.inf)
            top = w.amax(1, keepdim=True)
            e = torch.exp(w - torch.where(torch.isfinite(top), top, 0.0))
            tot = e.sum(1, keepdim=True)
            p = e / torch.where(tot > 0, tot, 1.0)
            o = p @ vv
            mag = (abs(scale) * (qq.abs() @ kk.abs().T) + (cap or 0.0) + abs(s) * d)
            dw = ((C + 1 + 8) * U * mag).amax(1, keepdim=True) + 4 * U * w.masked_fill(~seen, 0.0).abs().amax(1, True)
            dp = 2 * dw + (n + 8) * U
            o_b = (p * (dp + h + (n + 8) * U)) @ vv.abs() + step * o.abs() + tiny * (1 + vv.abs().sum(0, keepdim=True))
            out[rq, head], out_b[rq, head] = o, o_b
            if grad is None:
                continue
            go = grad[rq, head].double()
            gp = go @ vv.T
            D = (go * o).sum(1, keepdim=True)
            e_gp = (C + 2) * U * (go.abs() @ vv.abs().T)
            e_D = (go.abs() * o_b).sum(1, keepdim=True) + (C + 2) * U * (go.abs() * o.abs()).sum(1, keepdim=True)
            slack = 1 - (z / cap) ** 2 if cap else torch.ones_like(z)
            e_slack = 2 * (z / cap).abs() * (8 * U + dw / cap) + 2 * U if cap else torch.zeros_like(z)
            t = p * (gp - D) * slack
            t_b = p * ((gp - D).abs() * (slack * (dp + h + 8 * U) + e_slack) + slack * (e_gp + e_D)) + tiny
            gv[rk, head // G] += p.T @ go
            gv_b[rk, head // G] += (p * (dp + h + (n + 8) * U) + tiny).T @ go.abs()
            gq[rq, head] = t @ kk * scale
            gq_b[rq, head] = abs(scale) * ((t_b + (nk + 8) * U * t.abs()) @ kk.abs()) + step * gq[rq, head].abs() + tiny
            gk[rk, head // G] += t.T @ qq * scale
            gk_b[rk, head // G] += abs(scale) * ((t_b + (n + 8) * U * t.abs()).T @ qq.abs())
            if slope is not None:
                # sums of p, p gp and p gp d in float32, however they are grouped
                gs[head] -= (p * (gp - D) * d).sum()
                pd, pgp = (p * d).sum(1), (p * gp.abs()).sum(1)
                gs_b[head] += ((pd * pgp + (p * gp.abs() * d).sum(1)) * (2 * dp[:, 0] + (2 * nk + 16) * U)
                               + pd * (p * e_gp).sum(1) + (p * e_gp * d).sum(1)).sum()
                gs_b[head] += (nq + 8) * U * (pd * pgp).sum()
    r = {"out": (out, out_b)}
    if grad is not None:
        gk_b += step * gk.abs() + tiny
        gv_b += step * gv.abs() + tiny
        r |= {"q": (gq, gq_b), "k": (gk, gk_b), "v": (gv, gv_b)}
        if slope is not None:
            r["slope"] = (gs, gs_b + 1e-30)
    return r


def assert_within(name, got, value, bound):
    got = got.detach().double()
    assert bool(torch.isfinite(got).all()), f"{name}: not finite"
    over = (got - value).abs() - bound
    worst = float(over.max()) if over.numel() else -1.0
    assert worst <= 0.0, (f"{name}: {int((over > 0).sum())} of {over.numel()} outside their bound, worst by {worst:.3g} "
                          f"(bound there {float(bound.reshape(-1)[over.argmax()]):.3g})")
