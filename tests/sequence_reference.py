"""64-bit plain forms of the training LayerNorm and of sequence attention, with bounds on how far a
kernel that rounds where the documented types round may be from them.

A rounding to type t is off by at most u(t) = eps(t) / 2 of the value. The bounds count, element by
element: each rounding to the operands' type (P and dS before a matrix product, the output kept for the
backward pass, the results), and FP32 arithmetic as n u(fp32) of the sum of absolute terms for n
operations in a row."""

import math

import torch

U32 = 2.0 ** -24


def unit(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------ attention

def visible(batch, nq, nk, causal=False, prefix=None, documents=None, lengths=None):
    """[B, Nq, Nk] mask and [B, Nq] places, one query at a time."""
    keep = torch.zeros(batch, nq, nk, dtype=torch.bool)
    places = torch.zeros(batch, nq, dtype=torch.int64)
    for b in range(batch):
        n = nk if lengths is None else min(max(int(lengths[b]), 0), nk)
        pre = 0 if prefix is None else int(prefix if isinstance(prefix, int) else prefix[b])
        docs = None if documents is None else documents if documents.dim() == 1 else documents[b]
        for i in range(nq):
            p = n - nq + i
            places[b, i] = p
            if lengths is not None and p < 0:
                continue
            row = torch.arange(nk) < n
            if causal:
                row &= (torch.arange(nk) <= p) | (torch.arange(nk) < pre)
            if docs is not None:
                row &= (docs == docs[p]) & (docs[p] >= 0)
            keep[b, i] = row
    return keep, places


def attend(q, k, v, dout=None, *, causal=False, prefix=None, documents=None, lengths=None, softcap=None, slopes=None,
           scale=None):
    """Results and their bounds: {"out": (value, bound), "dq": ..., ...}, in 64 bits on the CPU."""
    dtype = q.dtype
    u = unit(dtype)
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    dout = None if dout is None else dout.detach().cpu().double()
    host = lambda t: t.cpu() if isinstance(t, torch.Tensor) else t                                    # noqa: E731
    B, H, nq, D = q.shape
    Hk, nk, Dv = k.shape[1], k.shape[2], v.shape[3]
    keep, places = visible(B, nq, nk, causal, host(prefix), host(documents), host(lengths))
    gap = (places[:, :, None] - torch.arange(nk)).abs().double()
    scale = D ** -0.5 if scale is None else scale
    res = {"out": [torch.zeros(B, H, nq, Dv, dtype=torch.float64) for _ in range(2)]}
    if dout is not None:
        for name, like in (("dq", q), ("dk", k), ("dv", v)):
            res[name] = [torch.zeros_like(like) for _ in range(2)]
        if slopes is not None:
            res["dslopes"] = [torch.zeros(H, dtype=torch.float64) for _ in range(2)]
    for b in range(B):
        for h in range(H):
            kv = h // (H // Hk)
            see = keep[b]
            clean = lambda t, rows: torch.where(rows[:, None], t, torch.zeros_like(t))               # noqa: E731
            rows, cols = see.any(1), see.any(0)
            qb, kb, vb = clean(q[b, h], rows), clean(k[b, kv], cols), clean(v[b, kv], cols)
            x = qb @ kb.T * scale
            c = softcap * torch.tanh(x / softcap) if softcap else x
            slope = 0.0 if slopes is None else float(slopes[h])
            s = c - slope * gap[b]
            P = torch.softmax(s.masked_fill(~see, -math.inf), -1).masked_fill(~see, 0.0)
            # Relative error of P: that of the scores (dot product, cap, distance, change of base)
            # against the row's largest one, and of the row's sum.
            es = (D + 8) * U32 * scale * (qb.abs() @ kb.abs().T) + 8 * U32 * (s.abs() + slope * gap[b])
            if softcap:
                es = es + softcap * (2.0 ** -21 if dtype == torch.bfloat16 else 8 * U32)
            es = torch.where(see, es, torch.zeros_like(es))
            eP = 2 * (es + es.amax(1, keepdim=True)) + (nk + 16) * U32
            out = P @ vb
            eout = (P * (eP + u + nk * U32)) @ vb.abs() + u * out.abs()
            res["out"][0][b, h], res["out"][1][b, h] = out, eout
            if dout is None:
                continue
            g = clean(dout[b, h], rows)
            dP = g @ vb.T
            delta = (g * out).sum(1, keepdim=True)
            edelta = (g.abs() * eout).sum(1, keepdim=True) + Dv * U32 * (g * out).abs().sum(1, keepdim=True)
            edP = Dv * U32 * (g.abs() @ vb.abs().T)
            dS = P * (dP - delta)
            bent = 1 - (c / softcap) ** 2 if softcap else torch.ones_like(c)
            ebent = 2.0 ** -20 if softcap else 0.0
            dX = dS * bent
            edX = P * ((edelta + edP + (dP - delta).abs() * (eP + u + 4 * U32)) * bent + (dP - delta).abs() * ebent)
            dq, dk, dv = dX @ kb * scale, dX.T @ qb * scale, P.T @ g
            res["dq"][0][b, h] = dq
            res["dq"][1][b, h] = ((edX + nk * U32 * dX.abs()) @ kb.abs()) * scale + u * dq.abs()
            n = nq * (H // Hk)
            res["dk"][0][b, kv] += dk
            res["dk"][1][b, kv] += ((edX + n * U32 * dX.abs()).T @ qb.abs()) * scale
            res["dv"][0][b, kv] += dv
            res["dv"][1][b, kv] += (P * (eP + u + n * U32)).T @ g.abs()
            if slopes is not None:
                res["dslopes"][0][h] -= (dS * gap[b]).sum()
                # Its sums are in FP32 throughout: P dP |.|, and P dP times P |.|.
                far, rel = (P * gap[b]).sum(1), eP.amax(1) + (nk + Dv + 8) * U32
                mass = (P * (g.abs() @ vb.abs().T) * gap[b]).sum(1) + (P * (g.abs() @ vb.abs().T)).sum(1) * far
                res["dslopes"][1][h] += (2 * rel * mass).sum()
    for name in ("dk", "dv"):
        if name in res:
            res[name][1] += u * res[name][0].abs()
    return {name: tuple(pair) for name, pair in res.items()}


# ------------------------------------------------------------------------------ LayerNorm

def norm(x, w, b, dy, eps, out_dtype):
    """{"y": (value, bound), "dx": ..., "dw": ..., "db": ...} for rows x [rows, C]."""
    ux, uy = unit(x.dtype), unit(out_dtype)
    uw, ub = (0.0 if t is None else unit(t.dtype) for t in (w, b))
    x, dy = x.detach().cpu().double(), dy.detach().cpu().double()
    rows, C = x.shape
    w = torch.ones(C, dtype=torch.float64) if w is None else w.detach().cpu().double().reshape(-1)
    b = torch.zeros(C, dtype=torch.float64) if b is None else b.detach().cpu().double().reshape(-1)
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = ((d * d).mean(1, keepdim=True) + eps).rsqrt()
    h = d * rstd
    # Sums over a row: up to 72 terms a lane (C / 256 of them beyond 16384 columns) and 10 joining steps.
    n = (max(72, C // 256) + 16) * U32
    ed = n * x.abs().mean(1, keepdim=True) + U32 * x.abs()
    # Variance: 2 |d| ed + (terms' sum); 1/deviation: half of its relative error.
    erel = ((2 * d.abs() * ed + ed * ed).mean(1, keepdim=True) * rstd * rstd + n) / 2 + 4 * U32
    eh = ed * rstd + h.abs() * erel + 2 * U32 * h.abs()
    y = h * w + b
    g = dy * w
    mg, mgh = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    dx = rstd * (g - mg - h * mgh)
    emgh = (g.abs() * eh).mean(1, keepdim=True) + n * (g * h).abs().mean(1, keepdim=True)
    edx = rstd * (n * g.abs().mean(1, keepdim=True) + eh * mgh.abs() + h.abs() * emgh
                  + 4 * U32 * (g.abs() + mg.abs() + (h * mgh).abs())) + dx.abs() * erel
    # Sums over rows: those of one lane, of the row groups, and of the workgroups in 16 slices.
    m = (rows // 1024 + 64 + 16 + 64 + 16) * U32 if rows > 16 else rows * U32 + 16 * U32
    dw, db = (dy * h).sum(0), dy.sum(0)
    return {"y": (y, w.abs() * eh + 2 * U32 * (y.abs() + b.abs()) + uy * y.abs()),
            "dx": (dx, edx + ux * dx.abs()),
            "dw": (dw, (dy.abs() * eh).sum(0) + m * (dy * h).abs().sum(0) + uw * dw.abs()),
            "db": (db, m * dy.abs().sum(0) + ub * db.abs())}


def check(got, want, what):
    """Every element within its bound (and of the same shape, finite)."""
    value, bound = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    if got.numel() == 0:
        return
    over = (got - value).abs() - bound * (1 + 1e-6) - 1e-37
    worst = float(((got - value).abs() / (bound + 1e-37)).max())
    print(f"[bound] {what}: at most {worst:.3f} of its bound", flush=True)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    assert float(over.max()) <= 0, f"{what}: {worst:.2f} times its bound at {int(over.argmax())}"
