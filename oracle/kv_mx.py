"""64-bit oracle of the 8- and 4-bit K/V cache and of decode attention with sinks (CPU)."""
from __future__ import annotations

import math

import torch

GROUP, PAGE = 32, 64
E_MIN = -116


def grid(fmt: str) -> torch.Tensor:
    """Values >= 0 of e2m1 or e4m3, ascending: code c holds grid[c]."""
    if fmt == "mxfp4":
        return torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
    vals = [m * 2.0**-9 for m in range(8)]
    vals += [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)]
    return torch.tensor(vals[:-1], dtype=torch.float64)


def group_exponent(amax: float, fmt: str) -> int:
    """The smallest integer e with amax <= (largest value + half a step) 2^e, in the kept range."""
    limit, e_max = (7.0, 125) if fmt == "mxfp4" else (464.0, 119)
    if amax == 0.0:
        return E_MIN
    e = math.frexp(amax)[1] - 12  # below any answer
    while amax > limit * 2.0**e:
        e += 1
    return min(max(e, E_MIN), e_max)


def hold(x: torch.Tensor, fmt: str) -> torch.Tensor:
    """The float64 values that a cache of `fmt` holds for x (..., hd)."""
    g = grid(fmt)
    out = torch.empty(x.shape, dtype=torch.float64)
    xs, os = x.double().reshape(-1, GROUP), out.view(-1, GROUP)
    for i, row in enumerate(xs):
        amax = row.abs().max()
        if not torch.isfinite(row).all():
            os[i] = math.nan
            continue
        s = 2.0 ** group_exponent(float(amax), fmt)
        dist = (row.abs()[:, None] / s - g).abs()
        best = dist.min(1, keepdim=True).values
        near = dist == best  # one value, or the two that a tie lies between: the even code
        code = torch.where(near.sum(1) == 2, near.int().argmax(1) + near.int().argmax(1) % 2, near.int().argmax(1))
        os[i] = torch.copysign(g[code] * s, row)
    return out


def support(pos: int, window: int, sinks: int, pages: list[int]) -> list[int]:
    """Attended tokens; the tokens of a page listed twice come twice."""
    ls = max(0, pos + 1 - window)
    se = min(sinks, ls)
    toks = list(range(se)) + list(range(ls, pos + 1))
    for pg in pages:
        toks += [t for t in range(pg * PAGE, pg * PAGE + PAGE) if se <= t < ls]
    return toks


def decode(q, k, v, toks, scale):
    """One sequence: q (Hq, hd), k, v (Hkv, T, hd) held values -> (out (Hq, hd), bound terms).

    The terms are, per output: sum_t p |v|, the largest sum_d |q k| of a row, the token count."""
    Hq, hd = q.shape
    G = Hq // k.shape[0]
    out, mag = torch.zeros(Hq, hd, dtype=torch.float64), torch.zeros(Hq, hd, dtype=torch.float64)
    big = torch.zeros(Hq, 1, dtype=torch.float64)
    for h in range(Hq):
        if not toks:
            continue
        kk, vv, qq = k[h // G, toks].double(), v[h // G, toks].double(), q[h].double()
        p = torch.softmax(kk @ qq * scale, 0)
        out[h], mag[h] = p @ vv, p @ vv.abs()
        big[h] = (kk.abs() @ qq.abs()).max() * abs(scale)
    return out, (mag, big, len(toks))
