"""Windowed attention with sinks, forward and gradients, against the 64-bit oracle and differences."""
import math

import pytest
import torch

from oracle import sink_attention as oracle

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
# unit roundoffs: of the type, and of P and dS as they enter the products
UNIT = {BF16: (2.0**-8, 2.0**-8), F32: (2.0**-24, 2.0**-23)}


def _inputs(B, Hq, Hkv, Tq, Tk, hd, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    # (B, H, T, hd) views of (B, T, H, hd) buffers, as a projection gives them
    return [torch.randn(B, T, H, hd, generator=g).to(dtype).transpose(1, 2)
            for T, H in ((Tq, Hq), (Tk, Hkv), (Tk, Hkv), (Tq, Hq))]


def _check(got, want, tol, names=("out", "dq", "dk", "dv")):
    for name, a, w, t in zip(names, got, want, tol):
        d = (a.double().cpu() - w).abs()
        # 1e-30: where nothing is attended both are exactly 0
        assert (d <= t + 1e-30).all(), (name, float((d / (t + 1e-30)).max()), int((d > t + 1e-30).sum()))


def _run(fsi, dev, q, k, v, dout, **kw):
    qd, kd, vd = (t.to(dev).requires_grad_() for t in (q, k, v))
    out = fsi.sink_window_attention(qd, kd, vd, **kw)
    grads = torch.autograd.grad(out, (qd, kd, vd), dout.to(dev))
    assert all(gr.dtype == q.dtype and gr.shape == t.shape for gr, t in zip(grads, (q, k, v)))
    return (out.detach(), *grads)


# (B, Hq, Hkv, Tq, Tk, window, sinks, lengths)
SHAPES = [
    (1, 1, 1, 1, 1, 1, 0, None),
    (1, 2, 1, 5, 5, 2, 1, None),
    (2, 4, 2, 64, 64, 64, 0, None),
    (1, 4, 2, 130, 130, 20, 3, None),
    (2, 3, 3, 77, 200, 33, 5, [200, 131]),
    (1, 4, 1, 300, 300, 64, 70, None),  # sinks over two tiles
    (2, 2, 2, 129, 129, 1, 1, [129, 0]),  # an empty sequence
    (1, 6, 2, 200, 200, 1000, 4, [150]),  # the window holds everything
    (1, 2, 2, 150, 150, 0, 90, None),  # sinks alone
    (1, 8, 2, 1, 333, 100, 4, None),  # one query
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd", [64, 128, 80])
@pytest.mark.parametrize("B,Hq,Hkv,Tq,Tk,window,sinks,lengths", SHAPES)
def test_values_and_gradients(fsi, dev, dtype, hd, B, Hq, Hkv, Tq, Tk, window, sinks, lengths):
    q, k, v, dout = _inputs(B, Hq, Hkv, Tq, Tk, hd, dtype, seed=Tk + hd)
    n = None if lengths is None else torch.tensor(lengths)
    scale = 1 / math.sqrt(hd)
    got = _run(fsi, dev, q, k, v, dout, window=window, sinks=sinks, lengths=None if n is None else n.to(dev))
    want, tol = oracle.attention(q, k, v, dout, window, sinks, n, scale, *UNIT[dtype])
    _check(got, want, tol)
    with torch.no_grad():  # the forward alone
        out = fsi.sink_window_attention(q.to(dev), k.to(dev), v.to(dev), window=window, sinks=sinks,
                                        lengths=None if n is None else n.to(dev))
    assert torch.equal(out, got[0])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd", [1, 16, 32, 40, 96, 200, 256])
def test_head_sizes(fsi, dev, dtype, hd):
    q, k, v, dout = _inputs(1, 2, 1, 70, 90, hd, dtype, seed=hd)
    got = _run(fsi, dev, q, k, v, dout, window=30, sinks=2, scale=0.3)
    _check(got, *oracle.attention(q, k, v, dout, 30, 2, None, 0.3, *UNIT[dtype]))


@pytest.mark.parametrize("hd", [20, 96, 200, 256])
def test_padded_heads(fsi, dev, hd, monkeypatch):
    """bf16 heads of other sizes, padded to the MFMA kernels' next size as large calls are."""
    from foveal_sparse_indexer_amd import sink_attention

    monkeypatch.setattr(sink_attention, "_PAD_WORK", 0)
    q, k, v, dout = _inputs(1, 8, 4, 600, 600, hd, BF16, seed=hd)
    got = _run(fsi, dev, q, k, v, dout, window=300, sinks=4)
    _check(got, *oracle.attention(q, k, v, dout, 300, 4, None, 1 / math.sqrt(hd), *UNIT[BF16]))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd", [64, 128])
def test_longer_rows(fsi, dev, dtype, hd):
    """Windows of several tiles with whole tiles inside, a ragged end and sinks far away."""
    q, k, v, dout = _inputs(1, 4, 2, 777, 777, hd, dtype, seed=7)
    got = _run(fsi, dev, q, k, v, dout, window=321, sinks=4)
    _check(got, *oracle.attention(q, k, v, dout, 321, 4, None, 1 / math.sqrt(hd), *UNIT[dtype]))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd,Hq,Hkv,Tq,Tk,window,sinks,lengths", [
    (64, 2, 1, 1500, 1500, 64, 70, None),  # sinks over two tiles
    (128, 3, 1, 1290, 1400, 100, 4, [1333]),  # fewer queries than keys, padded
    (80, 2, 2, 1217, 1217, 0, 5, None),
])
def test_sinks_seen_from_afar(fsi, dev, dtype, hd, Hq, Hkv, Tq, Tk, window, sinks, lengths):
    """Sink rows whose gradients come in several parts."""
    q, k, v, dout = _inputs(1, Hq, Hkv, Tq, Tk, hd, dtype, seed=Tq)
    n = None if lengths is None else torch.tensor(lengths)
    got = _run(fsi, dev, q, k, v, dout, window=window, sinks=sinks, lengths=None if n is None else n.to(dev))
    _check(got, *oracle.attention(q, k, v, dout, window, sinks, n, 1 / math.sqrt(hd), *UNIT[dtype]))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd", [64, 128, 48])
@pytest.mark.parametrize("Hq,Hkv,Tq,Tk,window,sinks,lengths", [
    (4, 1, 1, 2100, 2100, 0, None),  # one query, all keys
    (2, 1, 20, 1500, 1400, 70, [1490]),  # sinks and a long window
    (8, 1, 300, 300, 300, 3, None),  # one KV head for all
    (6, 2, 130, 1030, 1000, 4, [900]),  # no query inside the length
])
def test_few_rows_over_many_keys(fsi, dev, dtype, hd, Hq, Hkv, Tq, Tk, window, sinks, lengths):
    """Keys (query heads) cut into parts that are joined at the end."""
    q, k, v, dout = _inputs(1, Hq, Hkv, Tq, Tk, hd, dtype, seed=Tk)
    n = None if lengths is None else torch.tensor(lengths)
    got = _run(fsi, dev, q, k, v, dout, window=window, sinks=sinks, lengths=None if n is None else n.to(dev))
    _check(got, *oracle.attention(q, k, v, dout, window, sinks, n, 1 / math.sqrt(hd), *UNIT[dtype]))


@pytest.mark.parametrize("dtype,hd", [(BF16, 64), (BF16, 128), (BF16, 40), (F32, 64)])
def test_more_tiles_than_compute_units(fsi, dev, dtype, hd):
    """Enough heads for a workgroup on every compute unit: nothing but the sinks is cut."""
    q, k, v, dout = _inputs(2, 18, 9, 1000, 1000, hd, dtype, seed=hd)
    lengths = torch.tensor([1000, 950])
    got = _run(fsi, dev, q, k, v, dout, window=100, sinks=4, lengths=lengths.to(dev))
    _check(got, *oracle.attention(q, k, v, dout, 100, 4, lengths, 1 / math.sqrt(hd), *UNIT[dtype]))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_memory_behind_the_lengths_is_not_used(fsi, dev, dtype):
    q, k, v, dout = _inputs(2, 2, 1, 150, 150, 64, dtype, seed=3)
    lengths = torch.tensor([100, 1])
    want, tol = oracle.attention(q, k, v, dout, 40, 2, lengths, 0.125, *UNIT[dtype])
    for t in (q, k, v, dout):
        for b, n in enumerate(lengths.tolist()):
            t[b, :, n:] = math.nan
    got = _run(fsi, dev, q, k, v, dout, window=40, sinks=2, lengths=lengths.to(dev))
    _check(got, want, tol)
    for t in got:
        assert (t[0, :, 100:] == 0).all() and (t[1, :, 1:] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_hidden_keys_and_large_scores(fsi, dev, dtype):
    """Infinite and NaN keys where no query of the row sees them, and scores of thousands."""
    q, k, v, dout = _inputs(1, 2, 1, 100, 100, 64, dtype, seed=4)
    q *= 40
    want, tol = oracle.attention(q, k, v, dout, 10, 0, None, 1.0, *UNIT[dtype])
    got = _run(fsi, dev, q, k, v, dout, window=10, sinks=0, scale=1.0)
    _check(got, want, tol)
    k[0, 0, 50] = math.inf
    k[0, 0, 51] = math.nan
    out = fsi.sink_window_attention(q.to(dev), k.to(dev), v.to(dev), window=10, sinks=0, scale=1.0).cpu()
    for rows in (slice(0, 50), slice(61, 100)):
        d = (out[:, :, rows].double() - want[0][:, :, rows]).abs()
        assert (d <= tol[0][:, :, rows]).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd", [64, 80])
def test_strides_and_alignment(fsi, dev, dtype, hd):
    """Contiguous heads, expanded KV heads, rows of odd alignment and a transposed head_dim."""
    B, Hq, T = 2, 4, 70
    q, k, v, dout = _inputs(B, Hq, 2, T, T, hd, dtype, seed=5)
    scale = 1 / math.sqrt(hd)
    want, tol = oracle.attention(q, k, v, dout, 20, 3, None, scale, *UNIT[dtype])

    def odd(t):
        buf = torch.zeros(*t.shape[:3], hd + 3, dtype=dtype, device=dev)
        buf[..., 1:hd + 1] = t.to(dev)
        return buf[..., 1:hd + 1]

    def flipped(t):  # unit stride over T
        return t.to(dev).transpose(2, 3).contiguous().transpose(2, 3)

    for lay in (lambda t: t.to(dev).contiguous(), odd, flipped):
        qd, kd, vd = (lay(t).requires_grad_() for t in (q, k, v))
        out = fsi.sink_window_attention(qd, kd, vd, window=20, sinks=3)
        _check((out.detach(), *torch.autograd.grad(out, (qd, kd, vd), lay(dout))), want, tol)
    # one KV head expanded to two: its gradients are summed by autograd
    k1, v1 = k[:, :1], v[:, :1]
    want, tol = oracle.attention(q, k1, v1, dout, 20, 3, None, scale, *UNIT[dtype])
    kd, vd, qd = (t.to(dev).requires_grad_() for t in (k1, v1, q))
    out = fsi.sink_window_attention(qd, kd.expand(-1, 2, -1, -1), vd.expand(-1, 2, -1, -1), window=20, sinks=3)
    grads = torch.autograd.grad(out, (qd, kd, vd), dout.to(dev))
    u = UNIT[dtype][0]  # each of the two heads' gradients is rounded, and their sum
    slack = [tol[0], tol[1]] + [t + 3 * u * (w.abs() + t) + u * w.abs().amax() for t, w in zip(tol[2:], want[2:])]
    _check((out.detach(), *grads), want, slack)


def test_gradients_match_differences(fsi, dev):
    q, k, v, dout = (t.to(dev) for t in _inputs(1, 2, 1, 20, 33, 32, F32, seed=6))
    args = [t.clone().requires_grad_() for t in (q, k, v)]

    def loss(*a):
        return (fsi.sink_window_attention(*a, window=9, sinks=2).double() * dout.double()).sum()

    grads = torch.autograd.grad(loss(*args), args)
    g = torch.Generator(device=dev).manual_seed(0)
    for i in range(3):
        d = torch.randn(args[i].shape, device=dev, generator=g)
        step, vals = 1e-2, []
        with torch.no_grad():
            for sgn in (1, -1):
                a = list(args)
                a[i] = args[i] + sgn * step * d
                vals.append(loss(*a))
        diff = (vals[0] - vals[1]).item() / (2 * step)
        exact = (grads[i].double() * d.double()).sum().item()
        # third derivatives: step^2 of a loss whose terms are of the size of the gradient
        assert abs(diff - exact) <= 2e-3 * (abs(exact) + (grads[i].double() * d.double()).abs().sum().item())


def test_refusals(fsi, dev):
    x = torch.randn(1, 4, 8, 64, device=dev)
    kv = x[:, :2]
    f = fsi.sink_window_attention
    with pytest.raises(TypeError):
        f(x, kv.to(BF16), kv, window=2)
    with pytest.raises(TypeError):
        f(x.half(), kv.half(), kv.half(), window=2)
    for bad in ((x, x[:, :3], x[:, :3]), (x, kv, kv[:, :, :5]), (x, kv[:, :, :5], kv[:, :, :5]),
                (x, kv[..., :32], kv[..., :32]), (x[0], kv, kv)):
        with pytest.raises(ValueError):
            f(*bad, window=2)
    with pytest.raises(ValueError):
        f(x, kv, kv, window=-1)
    with pytest.raises(ValueError):
        f(x, kv, kv, window=2, sinks=-1)
    with pytest.raises(ValueError, match="lengths"):
        f(x, kv, kv, window=2, lengths=torch.zeros(2, dtype=torch.int32, device=dev))
    with pytest.raises(ValueError, match="lengths"):
        f(x, kv, kv, window=2, lengths=torch.zeros(1, device=dev))
    with pytest.raises(ValueError, match="head_dim"):
        f(torch.zeros(1, 1, 2, 300, device=dev), torch.zeros(1, 1, 2, 300, device=dev),
          torch.zeros(1, 1, 2, 300, device=dev), window=2)
    with pytest.raises(RuntimeError):
        f(x, kv.cpu(), kv, window=2)
    assert tuple(f(x[:, :, :0], kv, kv, window=2).shape) == (1, 4, 0, 64)
    xg = x.clone().requires_grad_()
    gq, = torch.autograd.grad(f(xg, kv, kv, window=2).sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):  # once differentiable
        torch.autograd.grad(gq.sum(), xg)


def test_empty_query_gradients(fsi, dev):
    q = torch.zeros(1, 2, 0, 64, device=dev, requires_grad=True)
    k = torch.randn(1, 1, 5, 64, device=dev, requires_grad=True)
    out = fsi.sink_window_attention(q, k, k, window=3)
    gk, = torch.autograd.grad(out.sum(), k)
    assert (gk == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_other_stream_and_replayed_graph(fsi, dev, dtype):
    """Forward and backward captured once and replayed with new inputs, and on another stream."""
    q, k, v, dout = (t.to(dev) for t in _inputs(2, 4, 2, 130, 130, 64, dtype, seed=8))
    leaves = [t.requires_grad_() for t in (q, k, v)]

    def step(args):
        out = fsi.sink_window_attention(*args, window=50, sinks=3)
        return (out.detach(), *torch.autograd.grad(out, args, dout))

    want = [t.clone() for t in step(leaves)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step([t.detach().clone().requires_grad_() for t in leaves])
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    held_in = [t.detach().clone().requires_grad_() for t in leaves]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(held_in)
    for i in range(3):
        with torch.no_grad():
            held_in[0].copy_(leaves[0] * (1 + i))
        graph.replay()
        torch.cuda.synchronize()
        res = [t.clone() for t in held]
        for a, b in zip(res, step([t.detach().clone().requires_grad_() for t in held_in])):
            assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", [None, "mxfp8", "mxfp4"])
def test_prompt_then_tokens(fsi, dev, fmt):
    """A layer's use: the prompt by windowed attention, its K / V into the cache, then token by
    token over the cache; over bf16 pages the tokens' outputs are those of the whole prompt."""
    B, Hq, Hkv, hd, T, n0, W, S = 2, 4, 2, 64, 180, 150, 40, 3
    q, k, v, _ = (t.to(dev) for t in _inputs(B, Hq, Hkv, T, T, hd, BF16, seed=9))
    cache = fsi.FovealKVCache(B, T, Hkv, hd, 16, 64, dev, BF16, kv_format=fmt)
    with torch.no_grad():
        whole = fsi.sink_window_attention(q, k, v, window=W, sinks=S)
        prompt = fsi.sink_window_attention(q[:, :, :n0], k[:, :, :n0], v[:, :, :n0], window=W, sinks=S)
        assert torch.equal(prompt, whole[:, :, :n0])
        cache.load_dense(k[:, :, :n0], v[:, :, :n0])
        for t in range(n0, T):
            cache.load_dense(k[:, :, t:t + 1], v[:, :, t:t + 1], start=t)
            tok = fsi.decode_attention(q[:, :, t], cache, pos=t, window=W, remote_pages=None, remote_counts=None,
                                       scale=1 / math.sqrt(hd), sinks=S)
            kd, vd = cache.to_dense(t + 1)
            # the same keys and values through the prompt's operator: one query at the end
            ref = fsi.sink_window_attention(q[:, :, t:t + 1], kd, vd, window=W, sinks=S)[:, :, 0]
            want, tol = oracle.attention(q[:, :, t:t + 1].cpu(), kd.cpu(), vd.cpu(), torch.zeros(B, Hq, 1, hd), W, S,
                                         None, 1 / math.sqrt(hd), *UNIT[BF16])
            for got in (tok, ref):
                assert ((got.double().cpu() - want[0][:, :, 0]).abs() <= tol[0][:, :, 0]).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd", [64, 80, 128, 256])
@pytest.mark.parametrize("Hq,Hkv,Tq,Tk,window,sinks", [
    (2, 1, 1, 1, 1, 0), (3, 3, 1, 1, 9, 4), (4, 2, 100, 130, 1, 0), (4, 2, 100, 130, 0, 1), (2, 2, 300, 300, 1, 0),
])
def test_a_single_key_has_no_score_gradient(fsi, dev, dtype, hd, Hq, Hkv, Tq, Tk, window, sinks):
    """Softmax over one key is 1 whatever its score: dq and dk are 0 to the bit."""
    q, k, v, dout = _inputs(2, Hq, Hkv, Tq, Tk, hd, dtype, seed=hd + Tq)
    got = _run(fsi, dev, q * 3, k, v, dout * 100, window=window, sinks=sinks)
    assert (got[1] == 0).all() and (got[2] == 0).all()
    _check(got, *oracle.attention(q * 3, k, v, dout * 100, window, sinks, None, 1 / math.sqrt(hd), *UNIT[dtype]))


@pytest.mark.parametrize("hd", [64, 80, 128])
def test_the_output_is_kept_to_sixteen_bits_for_the_backward(fsi, dev, hd):
    """out and what rounding took from it: at most half a step, which is at most 2^-8 of out (rounding
    the remainder itself may bring it to exactly half a step, so that their sum need not round to out),
    and where P is not rounded (80) the sum is the value to 2^-16 of it and the result's fp32 error."""
    q, k, v, dout = _inputs(2, 4, 2, 150, 150, hd, BF16, seed=hd)
    out, lse, lo = torch.ops.fsi.sink_window_attention(
        q.to(dev), k.to(dev), v.to(dev), None, 40, 3, 1 / math.sqrt(hd), True)
    both = out.double() + lo.double()
    assert (lo.double().abs() <= 2.0**-8 * out.double().abs()).all() and (lo != 0).any()
    if hd == 80:
        want, _ = oracle.attention(q, k, v, dout, 40, 3, None, 1 / math.sqrt(hd), *UNIT[BF16])
        _, tol = oracle.attention(q, k, v, dout, 40, 3, None, 1 / math.sqrt(hd), *UNIT[F32])
        assert ((both.cpu() - want[0]).abs() <= tol[0] + 2.0**-16 * want[0].abs()).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("scale", [0.0, -0.2])
def test_scales_of_either_sign(fsi, dev, dtype, scale):
    q, k, v, dout = _inputs(1, 4, 2, 130, 130, 64, dtype, seed=12)
    got = _run(fsi, dev, q, k, v, dout, window=50, sinks=3, scale=scale)
    _check(got, *oracle.attention(q, k, v, dout, 50, 3, None, scale, *UNIT[dtype]))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_offsets_beyond_32_bits(fsi, dev, dtype):
    """Rows 2^21 elements apart in one buffer of more than 2^31, and sequences 2^31 apart: as their copies."""
    big = torch.zeros((1 << 31) + (1 << 23), dtype=dtype, device=dev)
    far = big.as_strided((1, 2, 1024, 64), (0, 64, 1 << 21, 1))
    seqs = big.as_strided((2, 2, 100, 64), (1 << 31, 64, 256, 1), 128)
    g = torch.Generator().manual_seed(15)
    for view in (far, seqs):
        B, H, T, hd = view.shape
        x = torch.randn(B, H, T, hd, generator=g).to(dtype).to(dev)
        view.copy_(x)
        q, _, _, dout = (t.to(dev) for t in _inputs(B, 4, H, T, T, hd, dtype, seed=T))
        got, want = [], []
        for kv, res in ((view, got), (x, want)):
            leaves = [t.detach().requires_grad_() for t in (q, kv, kv)]
            out = fsi.sink_window_attention(*leaves, window=70, sinks=3)
            res += [out.detach(), *torch.autograd.grad(out, leaves, dout)]
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_two_backwards_at_once(fsi, dev, dtype):
    """Calls on two streams at once, and graphs of them replayed on two, have workspaces of their own."""
    sets = [[t.to(dev) for t in _inputs(1, 8, 2, 64, 2000, 64, dtype, seed=s)] for s in (1, 2)]

    def step(q, k, v, dout):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = fsi.sink_window_attention(*leaves, window=1500, sinks=70)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

    want = [step(*s) for s in sets]
    graphs, held = [], []
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(step(*s))
    streams = [torch.cuda.Stream() for _ in sets]
    for i in range(6):
        got = held
        if i % 2:
            got = [None, None]
        for j, st in enumerate(streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                if i % 2:
                    got[j] = step(*sets[j])
                else:
                    graphs[j].replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
