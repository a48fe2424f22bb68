"""The 64-bit oracles of the 8- and 4-bit cache and of windowed attention with sinks against
hand-made values, torch's own formats and finite differences (CPU)."""
import math

import pytest
import torch

from oracle import kv_mx, sink_attention


def test_grids_are_the_element_formats():
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(kv_mx.grid("mxfp8"), codes)
    assert kv_mx.grid("mxfp4").tolist() == [0, 0.5, 1, 1.5, 2, 3, 4, 6]


@pytest.mark.parametrize("fmt,limit,top", [("mxfp4", 7.0, 6.0), ("mxfp8", 464.0, 448.0)])
def test_scale_keeps_the_largest_within_half_a_step(fmt, limit, top):
    x = torch.zeros(32, dtype=torch.float64)
    x[5] = limit  # exactly at the limit: clamped, scale 1
    assert kv_mx.hold(x, fmt)[5] == top
    x[5] = math.nextafter(limit, 1e9)
    assert kv_mx.hold(x, fmt)[5] == limit + (1 if fmt == "mxfp4" else 16)  # 2 * the next scale's grid


def test_ties_go_to_even_codes():
    x = torch.zeros(32)
    x[:9] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -2.5])
    assert kv_mx.hold(x, "mxfp4")[:9].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, -2]


def test_not_finite_group_and_neighbours():
    x = torch.ones(2, 64)
    x[0, 3], x[1, 40] = math.inf, math.nan
    y = kv_mx.hold(x, "mxfp8")
    assert torch.isnan(y[0, :32]).all() and torch.isnan(y[1, 32:]).all()
    assert (y[0, 32:] == 1).all() and (y[1, :32] == 1).all()


def test_support_is_a_union():
    toks = kv_mx.support(pos=300, window=100, sinks=70, pages=[0, 1, 3])
    assert sorted(toks) == list(range(0, 128)) + list(range(192, 301))
    assert kv_mx.support(pos=5, window=100, sinks=4, pages=[]) == list(range(6))
    assert kv_mx.support(pos=5, window=0, sinks=0, pages=[]) == []


def test_attention_gradients_match_differences():
    g = torch.Generator().manual_seed(0)
    B, Hq, Hkv, Tq, Tk, hd = 1, 2, 1, 5, 9, 3
    q, dout = (torch.randn(B, Hq, Tq, hd, generator=g, dtype=torch.float64) for _ in range(2))
    k, v = (torch.randn(B, Hkv, Tk, hd, generator=g, dtype=torch.float64) for _ in range(2))
    lengths = torch.tensor([8])

    def run(q, k, v):
        return sink_attention.attention(q, k, v, dout, 3, 2, lengths, 0.7, 0.0, 0.0)[0]

    grads = run(q, k, v)[1:]
    for i, t in enumerate((q, k, v)):
        for idx in [(0, 0, 1, 0), (0, 0, 3, 2), (0, 0, 4, 1)]:
            step = torch.zeros_like(t)
            step[idx] = 1e-6
            args = [q, k, v]
            args[i] = t + step
            hi = (run(*args)[0] * dout).sum()
            args[i] = t - step
            lo = (run(*args)[0] * dout).sum()
            assert abs((hi - lo) / 2e-6 - grads[i][idx]) < 1e-8
