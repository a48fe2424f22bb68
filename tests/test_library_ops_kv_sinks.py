"""torch.library registration of the 8- and 4-bit cache, decode attention with sinks and windowed
attention with sinks: fake shapes on the CPU, opcheck and compiled graphs on the GPU."""
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

BF16 = torch.bfloat16


def _fake(*shape, dtype=BF16):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def test_registered_and_fake_shapes(fsi):
    ops = torch.ops.fsi
    have = set(dir(ops))
    assert {"kv_mx_write", "kv_mx_read", "decode_attention_sinks", "sink_window_attention",
            "sink_window_attention_bwd"} <= have
    with FakeTensorMode():
        pool, table = _fake(10, 2 * 4352, dtype=torch.uint8), _fake(4, 10, dtype=torch.int32)
        k, v = ops.kv_mx_read(pool, pool, table, 2, 2, 77, 128, 10, 10, 0)
        assert k.shape == v.shape == (4, 2, 77, 128) and k.dtype == torch.float32
        assert ops.kv_mx_write(_fake(4, 2, 7, 128), _fake(4, 2, 7, 128), 2, None, 3, table, 10, 10, pool, pool) is None
        q3 = _fake(4, 8, 128)
        o = ops.decode_attention_sinks(q3, pool, pool, 2, table, 10, 10, 2, None, 70, 64, 4, None, None, 0, 0.1)
        assert o.shape == q3.shape and o.dtype == BF16
        q, kk = _fake(2, 8, 100, 64), _fake(2, 2, 130, 64)
        o, lse, lo = ops.sink_window_attention(q, kk, kk, None, 30, 4, 0.125, True)
        assert o.shape == q.shape and o.transpose(1, 2).is_contiguous() and lse.shape == (2, 8, 100)
        assert lo.shape == o.shape and lo.stride() == o.stride()
        assert ops.sink_window_attention(q, kk, kk, None, 30, 4, 0.125, False)[1].numel() == 0
        grads = ops.sink_window_attention_bwd(q, kk, kk, o, lo, o, lse, None, 30, 4, 0.125)
        assert [g.shape for g in grads] == [q.shape, kk.shape, kk.shape] and all(g.is_contiguous() for g in grads)


def _randn(*shape, seed, dtype=BF16):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


def _held(fsi, dev, fmt, B=2, T=150, H=2, hd=64, dtype=BF16):
    c = fsi.FovealKVCache(B, T, H, hd, 16, 64, dev, dtype, kv_format=fmt)
    c.load_dense(_randn(B, H, T, hd, seed=1, dtype=dtype), _randn(B, H, T, hd, seed=2, dtype=dtype))
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(5))
def test_opcheck(fsi, dev, i):
    ops = torch.ops.fsi
    c = _held(fsi, dev, "mxfp4")
    q, kv = _randn(2, 4, 70, 64, seed=3), _randn(2, 2, 90, 64, seed=4)
    out, lse, lo = ops.sink_window_attention(q, kv, kv, None, 30, 4, 0.125, True)
    op, args = [
        (ops.kv_mx_write, (_randn(2, 2, 5, 64, seed=5), _randn(2, 2, 5, 64, seed=6), 2, None, 9, c.page_table,
                           c.max_pages, c.n_phys_pages, c.k_cache, c.v_cache)),
        (ops.kv_mx_read, (c.k_cache, c.v_cache, c.page_table, 2, 2, 100, 64, c.max_pages, c.n_phys_pages, 1)),
        (ops.decode_attention_sinks, (_randn(2, 4, 64, seed=7), c.k_cache, c.v_cache, 2, c.page_table, c.max_pages,
                                      c.n_phys_pages, 2, None, 120, 30, 4, None, None, 0, 0.125)),
        (ops.sink_window_attention, (q, kv, kv, torch.tensor([90, 80], dtype=torch.int32, device=dev), 30, 4, 0.125,
                                     True)),
        (ops.sink_window_attention_bwd, (q, kv, kv, out, lo, _randn(2, 4, 70, 64, seed=8), lse, None, 30, 4, 0.125)),
    ][i]
    torch.library.opcheck(op, args, test_utils=("test_schema", "test_faketensor", "test_aot_dispatch_dynamic"))


@pytest.mark.gpu
def test_write_is_seen_by_autograd(fsi, dev):
    """A write marks the pools as changed, through the launch and through the dispatcher alike."""
    c = _held(fsi, dev, "mxfp8")
    before = c.k_cache._version
    c.load_dense(_randn(2, 2, 1, 64, seed=3), _randn(2, 2, 1, 64, seed=4), start=9)
    assert c.k_cache._version > before
    k = c.to_dense(10)[0]
    x = _randn(2, 2, 1, 64, seed=3).requires_grad_()  # the dispatcher's way
    before = c.k_cache._version
    c.load_dense(x, x, start=9)
    assert c.k_cache._version > before
    assert torch.equal(c.to_dense(10)[0], k)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [None, "mxfp8", "mxfp4"])
def test_compiled_step_matches_eager(fsi, dev, fmt):
    c = _held(fsi, dev, fmt)

    def step(q, k, v):
        p = fsi.sink_window_attention(q, k, v, window=20, sinks=2)
        t = fsi.decode_attention(p[:, :, -1], c, pos=140, window=50, remote_pages=None, remote_counts=None,
                                 scale=1 / math.sqrt(64), sinks=3)
        return p, t

    q, k = _randn(2, 4, 40, 64, seed=5), _randn(2, 2, 40, 64, seed=6)
    with torch.no_grad():
        want = step(q, k, k)
        got = torch.compile(step, backend="aot_eager", fullgraph=True)(q, k, k)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_compiled_training_matches_eager(fsi, dev):
    def loss(q, k, v):
        return fsi.sink_window_attention(q, k, v, window=20, sinks=2).float().square().sum()

    args = [_randn(2, 4, 40, 64, seed=5).requires_grad_(), _randn(2, 2, 40, 64, seed=6).requires_grad_(),
            _randn(2, 2, 40, 64, seed=7).requires_grad_()]
    want = torch.autograd.grad(loss(*args), args)
    got = torch.autograd.grad(torch.compile(loss, backend="aot_eager", fullgraph=True)(*args), args)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
