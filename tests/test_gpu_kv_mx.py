"""K/V cache held in 8 and 4 bits, and decode attention over it (and over bf16 pages with sinks),
against the 64-bit oracle."""
import math

import pytest
import torch

from oracle import kv_mx

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
FORMATS = ["mxfp4", "mxfp8"]


def _cache(fsi, dev, B, T, H, hd, dtype, fmt, permute=True, extra=0):
    n = -(-T // 64)
    g = torch.Generator().manual_seed(B * 1000 + T)
    table = torch.randperm(B * n + extra, generator=g)[:B * n].to(torch.int32).view(B, n) if permute else None
    return fsi.FovealKVCache(B, T, H, hd, 16, 64, dev, dtype, n_phys_pages=B * n + extra if permute else None,
                             page_table=table, kv_format=fmt)


def _held(x, fmt):
    return x.double() if fmt is None else kv_mx.hold(x, fmt)


# (B, Hkv, hd, tokens, start): one token, one group over a page edge, whole pages, ragged ones
WRITES = [(1, 1, 64, 1, 0), (2, 3, 96, 1, 63), (2, 2, 128, 130, 5), (1, 2, 256, 64, 64), (3, 1, 64, 200, 0)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,H,hd,n,start", WRITES)
def test_write_read_is_the_nearest_value(fsi, dev, fmt, dtype, B, H, hd, n, start):
    g = torch.Generator().manual_seed(n + hd)
    k = (torch.randn(B, H, n, hd, generator=g) * torch.exp(torch.randn(B, H, n, 1, generator=g) * 8)).to(dtype)
    v = torch.randn(B, H, n, hd, generator=g).to(dtype)
    k[0, 0, 0, :32] = 0
    # values at borders: ties, the clamped range, subnormal results
    v[0, 0, 0, :8] = torch.tensor([7.0, 5.0, 2.5, 3.5, 0.25, 0.75, -6.5, 1.25]).to(dtype)
    c = _cache(fsi, dev, B, start + n + 3, H, hd, dtype, fmt, extra=2)
    c.load_dense(k.to(dev), v.to(dev), start=start)
    ko, vo = c.to_dense(start + n)
    assert ko.dtype == dtype and tuple(ko.shape) == (B, H, start + n, hd)
    for got, x in ((ko, k), (vo, v)):
        assert torch.equal(got[:, :, start:].double().cpu(), kv_mx.hold(x, fmt))
        assert (got[:, :, :start] == 0).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_extremes(fsi, dev, fmt):
    """Groups of infinities, NaN, the type's largest and smallest values and zeros."""
    x = torch.ones(1, 1, 9, 64)
    x[0, 0, 0, 3], x[0, 0, 1, 40], x[0, 0, 2, 0] = math.inf, math.nan, -math.inf
    x[0, 0, 3] = torch.finfo(BF16).max
    x[0, 0, 4] = torch.finfo(F32).max
    x[0, 0, 5] = torch.finfo(F32).tiny
    x[0, 0, 6] = 1e-45  # the smallest subnormal
    x[0, 0, 7] = -torch.finfo(F32).max
    x[0, 0, 8] = torch.linspace(-2.0**-112, 2.0**-113, 64)
    c = _cache(fsi, dev, 1, 9, 1, 64, F32, fmt)
    c.load_dense(x.to(dev), x.to(dev))
    want = kv_mx.hold(x, fmt)
    for got in c.to_dense(9):
        got = got.double().cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


@pytest.mark.parametrize("fmt", FORMATS)
def test_write_leaves_other_tokens(fsi, dev, fmt):
    """A rewrite of some tokens changes those alone; strided and offset operands are read in place."""
    g = torch.Generator().manual_seed(3)
    B, H, hd, n = 2, 2, 128, 150
    c = _cache(fsi, dev, B, n, H, hd, BF16, fmt)
    k, v = (torch.randn(B, H, n, hd, generator=g).to(BF16).to(dev) for _ in range(2))
    c.load_dense(k, v)
    before = [t.clone() for t in c.to_dense(n)]
    wide = torch.randn(B, 9, H, 2 * hd + 2, generator=g).to(BF16).to(dev)
    k2 = wide[..., 1:1 + hd].transpose(1, 2)  # rows of odd alignment
    v2 = wide[..., hd + 1:2 * hd + 1].transpose(1, 2)
    c.load_dense(k2, v2, start=60)
    for got, old, new in zip(c.to_dense(n), before, (k2, v2)):
        assert torch.equal(got[:, :, :60], old[:, :, :60]) and torch.equal(got[:, :, 69:], old[:, :, 69:])
        assert torch.equal(got[:, :, 60:69].double().cpu(), kv_mx.hold(new.cpu(), fmt))


@pytest.mark.parametrize("fmt", FORMATS)
def test_write_positions_per_sequence(fsi, dev, fmt, monkeypatch):
    """Sequences at positions of their own; what falls outside the cache is skipped and reported."""
    g = torch.Generator().manual_seed(4)
    B, H, hd, n, T = 3, 1, 64, 4, 70
    c = _cache(fsi, dev, B, T, H, hd, F32, fmt)
    k, v = (torch.randn(B, H, n, hd, generator=g) for _ in range(2))
    starts = [62, 0, 126]  # the last one's tail lies behind the two pages
    c.load_dense(k.to(dev), v.to(dev), start=torch.tensor(starts, device=dev))
    ko, vo = c.to_dense(128)
    for b, s in enumerate(starts):
        m = min(n, 128 - s)
        assert torch.equal(ko[b, :, s:s + m].double().cpu(), kv_mx.hold(k[b, :, :m], fmt))
        assert torch.equal(vo[b, :, s:s + m].double().cpu(), kv_mx.hold(v[b, :, :m], fmt))
        assert (ko[b, :, :s] == 0).all() and (ko[b, :, s + m:] == 0).all()
    from foveal_sparse_indexer_amd import _lib

    with pytest.raises(IndexError):
        _lib.raise_device_errors(dev, "write")
    _lib.raise_device_errors(dev, "write")  # reported once


def _decode_case(fsi, dev, fmt, dtype, B, Hq, Hkv, hd, T, pos, window, sinks, pages, seed=0, scale=None, poison=False):
    g = torch.Generator().manual_seed(seed)
    scale = 1 / math.sqrt(hd) if scale is None else scale
    k, v = (torch.randn(B, Hkv, T, hd, generator=g).to(dtype) for _ in range(2))
    q = torch.randn(B, Hq, hd, generator=g).to(dtype)
    c = _cache(fsi, dev, B, T, Hkv, hd, dtype, fmt)
    if poison:  # what lies behind a sequence's position is never used
        c.k_cache.fill_(0xFF if fmt else math.nan)
        c.v_cache.fill_(0xFF if fmt else math.nan)
        for b in range(B):
            n = pos[b] + 1
            one = c.page_table[b:b + 1]
            sub = fsi.FovealKVCache(1, T, Hkv, hd, 16, 64, dev, dtype, n_phys_pages=c.n_phys_pages, page_table=one,
                                    kv_format=fmt)
            sub.k_cache, sub.v_cache = c.k_cache, c.v_cache
            sub.load_dense(k[b:b + 1, :, :n].to(dev), v[b:b + 1, :, :n].to(dev))
    else:
        c.load_dense(k.to(dev), v.to(dev))
    cap = max([len(p) for p in pages] or [0])
    rp = rc = None
    if cap:
        rp = torch.full((B, cap), -1, dtype=torch.int32)
        for b, p in enumerate(pages):
            rp[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
        rp, rc = rp.to(dev), torch.tensor([len(p) for p in pages], dtype=torch.int32, device=dev)
    out = fsi.decode_attention(q.to(dev), c, pos=torch.tensor(pos, device=dev), window=window, remote_pages=rp,
                               remote_counts=rc, scale=scale, sinks=sinks)
    assert out.dtype == dtype and tuple(out.shape) == (B, Hq, hd)
    _check_decode(out, q, _held(k, fmt), _held(v, fmt), pos, window, sinks, pages, scale)


def _check_decode(out, q, k, v, pos, window, sinks, pages, scale):
    # P enters as 16 (bf16 out) or 24 bits; scores and sums are fp32 (bounds as in the oracle of
    # windowed attention); one rounding to the output's type
    dtype, hd, e = out.dtype, q.shape[-1], 2.0**-24
    u, u_p = (2.0**-8, 2.0**-16) if dtype == BF16 else (2.0**-24, 2.0**-23)
    for b in range(q.shape[0]):
        toks = kv_mx.support(pos[b], window, sinks, pages[b] if pages else [])
        want, (mag, big, n) = kv_mx.decode(q[b].cpu(), k[b], v[b], toks, scale)
        tol = u * want.abs() + (u_p + 2 * (hd + 4) * e * big + (2 * n + 8) * e) * mag
        bad = (out[b].double().cpu() - want).abs() > tol
        assert not bad.any(), (b, int(bad.sum()), float(((out[b].double().cpu() - want).abs() / tol).nan_to_num().max()))


# (dtype, B, Hq, Hkv, hd, T, pos, window, sinks, pages per sequence)
DECODES = [
    (BF16, 1, 1, 1, 64, 1, [0], 5, 0, []),  # one token
    (BF16, 2, 8, 2, 128, 200, [130, 5], 40, 3, []),
    (BF16, 3, 4, 4, 64, 330, [329, 64, 63], 64, 70, [[0, 2], [], [0]]),  # sinks inside a listed page
    (BF16, 1, 21, 1, 96, 150, [149], 1, 1, [[0]]),  # more query heads than one tile holds
    (BF16, 2, 6, 2, 256, 100, [99, 40], 1 << 30, 0, []),
    (F32, 2, 6, 2, 64, 260, [259, 100], 30, 4, [[1, 2], [0]]),
    (F32, 1, 5, 1, 96, 70, [69], 100, 0, []),
    (F32, 2, 3, 3, 128, 129, [128, 127], 0, 5, []),  # sinks alone
    (F32, 1, 16, 1, 256, 65, [64], 10, 2, []),
    (BF16, 2, 4, 2, 128, 700, [699, 3], 500, 0, [[0, 1], []]),
]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype,B,Hq,Hkv,hd,T,pos,window,sinks,pages", DECODES)
def test_decode_matches_the_definition(fsi, dev, fmt, dtype, B, Hq, Hkv, hd, T, pos, window, sinks, pages):
    _decode_case(fsi, dev, fmt, dtype, B, Hq, Hkv, hd, T, pos, window, sinks, pages)


@pytest.mark.parametrize("Hq,Hkv,hd,T,pos,window,sinks,pages", [
    (4, 2, 128, 200, [199, 66], 60, 4, []),
    (8, 1, 64, 330, [329, 10], 64, 70, [[0, 2], []]),
    (17, 1, 128, 130, [129, 0], 1, 1, []),
])
def test_decode_with_sinks_over_bf16_pages(fsi, dev, Hq, Hkv, hd, T, pos, window, sinks, pages):
    _decode_case(fsi, dev, None, BF16, 2, Hq, Hkv, hd, T, pos, window, sinks, pages)


@pytest.mark.parametrize("fmt", [None, *FORMATS])
@pytest.mark.parametrize("window,sinks", [(1 << 20, 1), (33, 2), (1, 100)])
def test_memory_behind_the_position_is_not_used(fsi, dev, fmt, window, sinks):
    _decode_case(fsi, dev, fmt, BF16, 3, 4, 2, 128, 190, [100, 63, 0], window, sinks, [], poison=True)


@pytest.mark.parametrize("fmt", FORMATS)
def test_decode_of_a_long_context_in_many_parts(fsi, dev, fmt):
    """One sequence over many workgroups (partials and their merge), fp32 and bf16."""
    for dtype in (BF16, F32):
        _decode_case(fsi, dev, fmt, dtype, 1, 4, 1, 64, 5000, [4999], 1 << 20, 0, [], seed=2)


@pytest.mark.parametrize("fmt", FORMATS)
def test_no_token_gives_zero(fsi, dev, fmt):
    c = _cache(fsi, dev, 2, 64, 1, 64, BF16, fmt)
    c.load_dense(torch.ones(2, 1, 64, 64, device=dev, dtype=BF16), torch.ones(2, 1, 64, 64, device=dev, dtype=BF16))
    q = torch.ones(2, 2, 64, device=dev, dtype=BF16)
    out = fsi.decode_attention(q, c, pos=torch.tensor([3, -1], device=dev), window=0, remote_pages=None,
                               remote_counts=None, scale=1.0, sinks=0)
    assert (out == 0).all()
    out = fsi.decode_attention(q, c, pos=torch.tensor([3, -1], device=dev), window=2, remote_pages=None,
                               remote_counts=None, scale=1.0, sinks=0)
    assert (out[0] == 1).all() and (out[1] == 0).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_page_listed_twice_counts_twice(fsi, dev, fmt):
    _decode_case(fsi, dev, fmt, F32, 1, 2, 1, 64, 300, [299], 20, 3, [[1, 1, 0]])


@pytest.mark.parametrize("fmt", FORMATS)
def test_nan_scores_reach_their_sequence_only(fsi, dev, fmt):
    g = torch.Generator().manual_seed(8)
    k, v = (torch.randn(2, 1, 70, 64, generator=g) for _ in range(2))
    k[1, 0, 69, 5] = math.nan
    c = _cache(fsi, dev, 2, 70, 1, 64, F32, fmt)
    c.load_dense(k.to(dev), v.to(dev))
    q = torch.randn(2, 2, 64, generator=g)
    args = dict(window=1 << 20, remote_pages=None, remote_counts=None, scale=0.1)
    out = fsi.decode_attention(q.to(dev), c, pos=69, **args)
    assert torch.isnan(out[1]).all() and torch.isfinite(out[0]).all()
    # hidden, the NaN is not there
    out = fsi.decode_attention(q.to(dev), c, pos=68, **args)
    _check_decode(out, q, kv_mx.hold(k, fmt), kv_mx.hold(v, fmt), [68, 68], 1 << 20, 0, [], 0.1)


def test_bad_pages_are_skipped_and_reported(fsi, dev):
    from foveal_sparse_indexer_amd import _lib

    g = torch.Generator().manual_seed(9)
    k, v = (torch.randn(1, 1, 256, 64, generator=g).to(BF16) for _ in range(2))
    c = _cache(fsi, dev, 1, 256, 1, 64, BF16, "mxfp8")
    c.load_dense(k.to(dev), v.to(dev))
    q = torch.randn(1, 1, 64, generator=g).to(BF16)
    pages = torch.tensor([[1, 77, -5]], dtype=torch.int32, device=dev)
    out = fsi.decode_attention(q.to(dev), c, pos=255, window=10, remote_pages=pages,
                               remote_counts=torch.tensor([3], device=dev), scale=0.125, sinks=2)
    with pytest.raises(IndexError):
        _lib.raise_device_errors(dev, "decode")
    _check_decode(out, q, kv_mx.hold(k, "mxfp8"), kv_mx.hold(v, "mxfp8"), [255], 10, 2, [[1]], 0.125)
    # a position behind the table: reported, the tokens that are there attended
    out = fsi.decode_attention(q.to(dev), c, pos=torch.tensor([300], device=dev), window=10, remote_pages=None,
                               remote_counts=None, scale=0.125)
    with pytest.raises(IndexError):
        _lib.raise_device_errors(dev, "decode")
    assert torch.isfinite(out).all()


def test_decode_refusals(fsi, dev):
    c = _cache(fsi, dev, 2, 64, 1, 64, BF16, "mxfp4")
    q = torch.zeros(2, 1, 64, device=dev, dtype=BF16)
    args = dict(window=4, remote_pages=None, remote_counts=None, scale=1.0)
    with pytest.raises(RuntimeError, match="gradient"):
        fsi.decode_attention(q.clone().requires_grad_(), c, pos=0, **args)
    with pytest.raises(TypeError):
        fsi.decode_attention(q.float(), c, pos=0, **args)
    with pytest.raises(ValueError, match="positions"):
        fsi.decode_attention(q, c, pos=torch.zeros(3, device=dev), **args)
    with pytest.raises(IndexError):
        fsi.decode_attention(q, c, pos=64, **args)
    with pytest.raises(ValueError, match="sinks"):
        fsi.decode_attention(q, c, pos=0, sinks=-1, **args)
    with pytest.raises(ValueError, match="out"):
        fsi.decode_attention(q, c, pos=0, out=torch.zeros(2, 1, 32, device=dev, dtype=BF16), **args)
    with pytest.raises(ValueError, match="capacity"):
        fsi.decode_attention(q, c, pos=0, window=4, remote_pages=torch.zeros(1, 3, device=dev),
                             remote_counts=torch.zeros(2, device=dev), scale=1.0)
    dense = fsi.FovealKVCache(2, 64, 1, 64, 16, 64, dev, F32)
    with pytest.raises(ValueError, match="paged"):
        fsi.decode_attention(q.float(), dense, pos=0, sinks=2, **args)
    with pytest.raises(ValueError, match="bf16"):
        fsi.decode_step_attention(q, torch.zeros(2, 16, device=dev, dtype=BF16), c, pos=0, window=4, completed_pages=0,
                                  top_p=0.9, min_remote_blocks=0, max_remote_blocks=2, scale=1.0)


@pytest.mark.parametrize("fmt", FORMATS)
def test_other_stream_and_replayed_graph(fsi, dev, fmt):
    """Write, read back and decode captured once and replayed with new inputs, beside an eager call
    of the same cache on another stream."""
    g = torch.Generator().manual_seed(11)
    B, H, hd, T = 2, 2, 64, 300
    c = _cache(fsi, dev, B, T, H, hd, BF16, fmt)
    k, v = (torch.randn(B, H, T, hd, generator=g).to(BF16) for _ in range(2))
    kd, vd, q = k.to(dev), v.to(dev), torch.randn(B, 4, hd, generator=g).to(BF16).to(dev)
    pos = torch.tensor([299, 120], dtype=torch.int32, device=dev)

    def step():
        c.load_dense(kd, vd)
        o = fsi.decode_attention(q, c, pos=pos, window=1 << 20, remote_pages=None, remote_counts=None, scale=0.125)
        return o, *c.to_dense(T)

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(3):
        kd.copy_(k.to(dev) * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        res = [t.clone() for t in held]
        eager = step()
        for a, b in zip(res, eager):
            assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_module_decodes_from_a_held_cache(fsi, dev, fmt, dtype):
    """FovealSparseAttention.decode_step over a cache in 8 or 4 bits: the same routing and the
    attention of the values that the cache holds."""
    torch.manual_seed(5)
    m = fsi.FovealSparseAttention(256, 4, 2, head_dim=64, local_window_blocks=1, max_remote_pages=2,
                                  min_remote_pages=1).to(dev, dtype)
    T, B = 200, 2
    xs = torch.randn(B, T, 256, device=dev).to(dtype)
    with torch.no_grad():
        cache, plain = (m.init_kv_cache(B, 256, dev, f) for f in (fmt, None))
        assert cache.kv_format == fmt
        for t in range(T):
            x = xs[:, t:t + 1]
            out, info = m.decode_step(x, cache)
            # the same step over a cache of the model's type that holds the rounded values
            kd, vd = cache.to_dense(t + 1)
            m.decode_step(x, plain)
            if t % 37 == 0 or t == T - 1:
                q = m.q_proj(x).view(B, 4, 64)
                pages = info["selected_remote_pages"]
                att = []
                for b in range(B):
                    toks = kv_mx.support(t, m.local_window, 0, pages[b])
                    att.append(kv_mx.decode(q[b].cpu(), kd[b].cpu(), vd[b].cpu(), toks, m.scale)[0])
                att = torch.stack(att).to(dev, dtype).view(B, 1, 256)
                want = m.out_proj(att)
                if cache.completed_pages:
                    qi = m.indexer.compute_query_16d(x)
                    from foveal_sparse_indexer_amd.attention import decode_route

                    ctx = decode_route(qi, cache.kp_cache, cache.vp_cache, pos=t, page_size=64, local_window=64,
                                       completed_pages=cache.completed_pages, top_p=m.indexer.top_p,
                                       min_remote_blocks=1, max_remote_blocks=2, return_context=True)[2]
                    want = want + m.indexer.out_proj(ctx.view(B, 1, -1))
                # att differs by a rounding of the type: 256 products of it through out_proj's weights
                u = torch.finfo(dtype).eps / 2
                tol = 4 * u * (att.abs().float() @ m.out_proj.weight.abs().float().t() + want.abs().float()) + 1e-6
                assert ((out - want).abs().float() <= tol).all()


@pytest.mark.parametrize("fmt,hd,H,n_phys", [("mxfp8", 256, 2, 140000), ("mxfp4", 256, 4, 140000),
                                              (None, 128, 2, 140000)])
def test_pages_beyond_32_bit_offsets(fsi, dev, fmt, hd, H, n_phys):
    """Pools of more than 4 GiB: pages at their end are written, read and attended as those of a small one."""
    high = torch.tensor([[n_phys - 1, 3, n_phys - 2]], dtype=torch.int32)
    g = torch.Generator().manual_seed(13)
    k, v = (torch.randn(1, H, 180, hd, generator=g).to(BF16).to(dev) for _ in range(2))
    q = torch.randn(1, 2 * H, hd, generator=g).to(BF16).to(dev)
    got = []
    for n, table in ((n_phys, high), (8, torch.tensor([[7, 3, 6]], dtype=torch.int32))):
        c = fsi.FovealKVCache(1, 192, H, hd, 16, 64, dev, BF16, n_phys_pages=n, page_table=table, kv_format=fmt)
        assert n == 8 or c.k_cache.numel() * c.k_cache.element_size() > 1 << 32
        c.load_dense(k, v)
        o = fsi.decode_attention(q, c, pos=179, window=70, remote_pages=torch.tensor([[0]], device=dev),
                                 remote_counts=torch.tensor([1], device=dev), scale=1 / math.sqrt(hd), sinks=9)
        got.append((o, *c.to_dense(180)))
    for a, b in zip(*got):
        assert torch.equal(a, b) and a.abs().max() > 0


def test_two_graphs_replayed_side_by_side(fsi, dev):
    """Graphs captured on one stream and replayed on two at once have partials of their own."""
    g = torch.Generator().manual_seed(14)
    T, hd = 5000, 128
    c = _cache(fsi, dev, 1, T, 1, hd, BF16, "mxfp4")
    c.load_dense(*(torch.randn(1, 1, T, hd, generator=g).to(BF16).to(dev) for _ in range(2)))
    qs = [torch.randn(1, 8, hd, generator=g).to(BF16).to(dev) for _ in range(2)]

    def step(q):
        return fsi.decode_attention(q, c, pos=T - 1, window=1 << 20, remote_pages=None, remote_counts=None,
                                    scale=1 / math.sqrt(hd), sinks=4)

    want = [step(q) for q in qs]
    graphs, held = [], []
    for q in qs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(step(q))
    streams = [torch.cuda.Stream() for _ in qs]
    for _ in range(5):
        for gr, st in zip(graphs, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("start", [(1 << 32) + 3, -(1 << 32) + 3, (1 << 31) - 1, -(1 << 31)])
def test_start_positions_beyond_32_bits(fsi, dev, fmt, start):
    """Outside the cache, not wrapped into it."""
    from foveal_sparse_indexer_amd import _lib

    c = _cache(fsi, dev, 2, 64, 1, 64, F32, fmt)
    x = torch.ones(2, 1, 2, 64, device=dev)
    c.load_dense(x, x, start=torch.tensor([start, 5], device=dev))
    ko, vo = c.to_dense(64)
    assert (ko[0] == 0).all() and (vo[0] == 0).all() and (ko[1, :, 5:7] == 1).all() and int((ko[1] != 0).sum()) == 128
    with pytest.raises(IndexError):
        _lib.raise_device_errors(dev, "write")
