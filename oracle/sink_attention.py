"""64-bit oracle of attention over a sliding window and sinks, with its gradients (CPU), and
bounds on what rounding may change."""
from __future__ import annotations

import math

import torch


def visible(Tq, Tk, window, sinks, length):
    """(Tq, Tk) mask of the keys that each query sees."""
    p = torch.arange(Tk - Tq, Tk)[:, None]
    s = torch.arange(Tk)[None]
    return (s <= p) & ((s > p - window) | (s < sinks)) & (p < length) & (s < length)


def attention(q, k, v, dout, window, sinks, lengths, scale, u, u_p):
    """(out, dq, dk, dv) in float64 and a bound on each one's error, for operands of unit
    roundoff u whose P and dS enter the products with unit roundoff u_p.

    Bounds: a score of hd terms summed in fp32 is off by (hd + 4) 2^-24 sum |q k|, and P by twice
    that, relatively (numerator and denominator), plus (Tk + 8) 2^-24 for the sum and exp2; D is
    taken from the rounded output; sums over n terms in fp32 cost n 2^-24 of their magnitudes."""
    B, Hq, Tq, hd = q.shape
    Hkv, Tk = k.shape[1], k.shape[2]
    G, e = Hq // Hkv, 2.0**-24
    qd, kd, vd, gd = (t.double() for t in (q, k, v, dout))
    res = [torch.zeros_like(qd), torch.zeros_like(qd), torch.zeros_like(kd), torch.zeros_like(vd)]
    tol = [torch.zeros_like(t) for t in res]
    for b in range(B):
        ok = visible(Tq, Tk, window, sinks, Tk if lengths is None else int(lengths[b]))
        rows = ok.any(1)
        okk = ok.any(0)
        for h in range(Hq):
            # hidden memory may hold anything: it takes no part
            qq, gg = (torch.where(rows[:, None], t[b, h], 0.0) for t in (qd, gd))
            kk, vv = (torch.where(okk[:, None], t[b, h // G], 0.0) for t in (kd, vd))
            x = (qq @ kk.T * scale).masked_fill(~ok, -math.inf)
            x = torch.where(rows[:, None], x, 0.0)
            p = torch.where(ok, torch.softmax(x, 1), 0.0)
            o = p @ vv
            dd = (gg * o).sum(1, keepdim=True)
            dp = gg @ vv.T
            ds = p * (dp - dd)
            rel = 2 * (hd + 4) * e * abs(scale) * torch.where(ok, qq.abs() @ kk.abs().T, 0.0).amax(1, keepdim=True)
            rel = rel + (Tk + 8) * e
            o_err = (rel + u_p + Tk * e) * (p @ vv.abs())
            res[0][b, h], tol[0][b, h] = o, u * o.abs() + o_err
            d_err = (gg.abs() * (u * o.abs() + o_err)).sum(1, keepdim=True) + hd * e * (gg.abs() * o.abs()).sum(1, True)
            ds_err = (rel + u_p) * ds.abs() + p * (1 + rel) * (d_err + (hd + 2) * e * (gg.abs() @ vv.abs().T))
            res[1][b, h] = ds @ kk * scale
            tol[1][b, h] = u * res[1][b, h].abs() + abs(scale) * ((ds_err + Tk * e * ds.abs()) @ kk.abs())
            n = Tq * G * e
            res[2][b, h // G] += ds.T @ qq * scale
            tol[2][b, h // G] += abs(scale) * ((ds_err + n * ds.abs()).T @ qq.abs())
            res[3][b, h // G] += p.T @ gg
            tol[3][b, h // G] += ((rel + u_p + n) * p).T @ gg.abs()
    tol[2] += u * res[2].abs()
    tol[3] += u * res[3].abs()
    return res, tol
