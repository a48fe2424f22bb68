"""CPU checks of the 8- and 4-bit cache, decode attention with sinks and windowed attention:
argument errors come back from the host before any launch."""
import pytest
import torch

FMT8, FMT4 = 1, 2


def _ptr(n=1):
    return 4096 * n


def test_block_bytes(fsi):
    from foveal_sparse_indexer_amd import _lib

    f = _lib.lib().fsi_kv_mx_block_bytes
    assert f(128, FMT4) == 64 * (64 + 4) and f(128, FMT8) == 64 * (128 + 4)
    assert f(96, FMT4) == 64 * (48 + 3) and f(256, FMT8) == 64 * (256 + 8)
    assert f(80, FMT4) == 0 and f(128, 0) == 0 and f(0, FMT4) == 0


def test_write_and_read_errors(fsi):
    from foveal_sparse_indexer_amd import _lib

    L = _lib.lib()

    def write(k=_ptr(1), hd=128, B=1, H=2, n=3, dtype=1, fmt=FMT4, start=0, table=_ptr(3), pages=4, phys=4,
              pool=_ptr(4)):
        return L.fsi_kv_mx_write(k, _ptr(2), 1, 1, 1, 1, 1, 1, B, H, n, hd, dtype, fmt, None, start, table, pages, phys,
                                 pool, _ptr(5), None, None)

    assert write(fmt=0) == _lib.FSI_ERR_INVALID_ARG and write(fmt=3) == _lib.FSI_ERR_INVALID_ARG
    assert write(dtype=2) == _lib.FSI_ERR_DTYPE
    assert write(hd=80) == _lib.FSI_ERR_SHAPE and write(H=0) == _lib.FSI_ERR_SHAPE
    assert write(n=-1) == _lib.FSI_ERR_SHAPE and write(start=-1) == _lib.FSI_ERR_SHAPE
    assert write(pages=0) == _lib.FSI_ERR_SHAPE and write(pages=1 << 40) == _lib.FSI_ERR_SHAPE
    assert write(k=None) == _lib.FSI_ERR_INVALID_ARG and write(table=None) == _lib.FSI_ERR_INVALID_ARG
    assert write(pool=_ptr(4) + 4) == _lib.FSI_ERR_ALIGN
    assert write(n=0, k=None) == _lib.FSI_OK and write(B=0, k=None) == _lib.FSI_OK

    def read(fmt=FMT8, hd=64, n=5, dtype=0, out=_ptr(6)):
        return L.fsi_kv_mx_read(_ptr(1), _ptr(2), fmt, 1, 2, n, hd, _ptr(3), 4, 4, dtype, out, _ptr(7), None)

    assert read(fmt=0) == _lib.FSI_ERR_INVALID_ARG and read(dtype=3) == _lib.FSI_ERR_DTYPE
    assert read(hd=32) == _lib.FSI_ERR_SHAPE and read(out=None) == _lib.FSI_ERR_INVALID_ARG
    assert read(out=_ptr(6) + 2) == _lib.FSI_ERR_ALIGN and read(n=0, out=None) == _lib.FSI_OK


def test_decode_errors(fsi):
    from foveal_sparse_indexer_amd import _lib

    L = _lib.lib()

    def decode(q=_ptr(1), dtype=1, fmt=FMT4, pages=4, phys=4, pos=10, window=8, sinks=2, remote=None, cap=0, B=1, Hq=4,
               Hkv=2, hd=128, ws=None, nbytes=0):
        return L.fsi_decode_attn_sinks(q, dtype, _ptr(2), _ptr(3), fmt, _ptr(4), pages, phys, None, pos, window, sinks,
                                       remote, remote, cap, B, Hq, Hkv, hd, 1.0, _ptr(5), ws, nbytes, None, None)

    assert decode(fmt=5) == _lib.FSI_ERR_INVALID_ARG
    assert decode(dtype=2) == _lib.FSI_ERR_DTYPE and decode(dtype=0, fmt=0) == _lib.FSI_ERR_DTYPE
    assert decode(hd=96, fmt=0) == _lib.FSI_ERR_SHAPE and decode(hd=72) == _lib.FSI_ERR_SHAPE
    assert decode(Hq=5) == _lib.FSI_ERR_SHAPE and decode(sinks=-1) == _lib.FSI_ERR_SHAPE
    assert decode(window=-1) == _lib.FSI_ERR_SHAPE and decode(phys=0) == _lib.FSI_ERR_SHAPE
    assert decode(pos=256) == _lib.FSI_ERR_INDEX_RANGE and decode(pos=-1) == _lib.FSI_ERR_SHAPE
    assert decode(q=None) == _lib.FSI_ERR_INVALID_ARG and decode(cap=3) == _lib.FSI_ERR_INVALID_ARG
    assert decode(q=_ptr(1) + 8) == _lib.FSI_ERR_ALIGN
    big = dict(pages=1 << 20, phys=1 << 20, pos=1 << 25, window=1 << 26)
    need = L.fsi_decode_attn_sinks_workspace_size(1, 4, 2, 128, FMT4, 1 << 26, 2, 0, 1 << 20)
    assert need > 0 and decode(**big) == _lib.FSI_ERR_WORKSPACE
    assert decode(**big, ws=_ptr(6), nbytes=need - 1) == _lib.FSI_ERR_WORKSPACE
    assert decode(B=0, q=None) == _lib.FSI_OK


def test_sink_attention_errors(fsi):
    from foveal_sparse_indexer_amd import _lib

    L = _lib.lib()

    def fwd(q=_ptr(1), B=1, Hq=4, Hkv=2, Tq=3, Tk=5, hd=64, window=2, sinks=1, dtype=1):
        return L.fsi_sink_attn(q, 1, 1, 1, _ptr(2), 1, 1, 1, _ptr(3), 1, 1, 1, B, Hq, Hkv, Tq, Tk, hd, window, sinks,
                               None, 1.0, dtype, _ptr(4), 1, 1, 1, None, None, None, 0, None)

    def bwd(q=_ptr(1), Tq=3, Tk=5, hd=64, dtype=1, ws=None, nbytes=0, dk=_ptr(8)):
        return L.fsi_sink_attn_bwd(q, 1, 1, 1, _ptr(2), 1, 1, 1, _ptr(3), 1, 1, 1, _ptr(4), 1, 1, 1, None, _ptr(5),
                                   1, 1, 1,
                                   _ptr(6), 1, 4, 2, Tq, Tk, hd, 2, 1, None, 1.0, dtype, _ptr(7), dk, _ptr(9), ws,
                                   nbytes, None)

    assert fwd(dtype=2) == _lib.FSI_ERR_DTYPE and fwd(hd=257) == _lib.FSI_ERR_SHAPE and fwd(hd=0) == _lib.FSI_ERR_SHAPE
    assert fwd(Hq=3) == _lib.FSI_ERR_SHAPE and fwd(Tq=6) == _lib.FSI_ERR_SHAPE and fwd(Tq=-1) == _lib.FSI_ERR_SHAPE
    assert fwd(window=-1) == _lib.FSI_ERR_SHAPE and fwd(sinks=-1) == _lib.FSI_ERR_SHAPE
    assert fwd(Tk=1 << 31) == _lib.FSI_ERR_SHAPE and fwd(q=None) == _lib.FSI_ERR_INVALID_ARG
    assert fwd(Tq=0, q=None) == _lib.FSI_OK and fwd(B=0, q=None) == _lib.FSI_OK
    assert fwd(Tq=1, Tk=8192, window=8192) == _lib.FSI_ERR_WORKSPACE  # one query over many keys runs in parts
    assert L.fsi_sink_attn_workspace_size(1, 4, 2, 1, 8192, 64, 8192, 0) > 0
    assert bwd(dtype=3) == _lib.FSI_ERR_DTYPE and bwd(hd=300) == _lib.FSI_ERR_SHAPE
    assert bwd(q=None) == _lib.FSI_ERR_INVALID_ARG and bwd(dk=None) == _lib.FSI_ERR_INVALID_ARG
    assert bwd() == _lib.FSI_ERR_WORKSPACE


def test_cache_constructor(fsi):
    def make(**over):
        a = dict(batch_size=1, max_seq_len=128, num_kv_heads=2, head_dim=128, index_dim=16, page_size=64, device="cpu",
                 dtype=torch.bfloat16, kv_format="mxfp4")
        a.update(over)
        return fsi.FovealKVCache(**a)

    c = make()
    assert c.paged and c.kv_format == "mxfp4" and c.k_cache.dtype == torch.uint8
    assert tuple(c.k_cache.shape) == (2, 2 * 64 * 68) and c.kp_cache.dtype == torch.float32
    assert make(dtype=torch.float32, head_dim=96, kv_format="mxfp8").paged
    for bad in (dict(kv_format="int4"), dict(page_size=32), dict(head_dim=80), dict(paged=False)):
        with pytest.raises(ValueError):
            make(**bad)
    with pytest.raises(TypeError):
        make(dtype=torch.float16)
    with pytest.raises(RuntimeError, match="capacity"):
        c.load_dense(torch.zeros(1, 2, 129, 128, dtype=torch.bfloat16), torch.zeros(1, 2, 129, 128).bfloat16())
    with pytest.raises(ValueError, match="do not match"):
        c.load_dense(torch.zeros(1, 3, 1, 128).bfloat16(), torch.zeros(1, 3, 1, 128).bfloat16())
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        c.load_dense(torch.zeros(1, 2, 1, 128).bfloat16(), torch.zeros(1, 2, 1, 128).bfloat16())
    with pytest.raises(ValueError, match="start positions"):
        c.load_dense(torch.zeros(1, 2, 1, 128).bfloat16(), torch.zeros(1, 2, 1, 128).bfloat16(),
                     start=torch.zeros(2, dtype=torch.int32))
    for dt in (torch.float32, torch.bool):
        with pytest.raises(TypeError, match="integers"):
            c.load_dense(torch.zeros(1, 2, 1, 128).bfloat16(), torch.zeros(1, 2, 1, 128).bfloat16(),
                         start=torch.zeros(1, dtype=dt))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        c.to_dense(4)
    plain = make(kv_format=None)
    with pytest.raises(TypeError, match="kv_format"):
        plain.load_dense(torch.zeros(1, 2, 1, 128).bfloat16(), torch.zeros(1, 2, 1, 128).bfloat16(),
                         start=torch.zeros(1, dtype=torch.int32))


def test_python_ops_refuse_cpu_tensors(fsi):
    x = torch.randn(1, 2, 4, 64)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        fsi.sink_window_attention(x, x, x, window=2)
    c = fsi.FovealKVCache(1, 64, 2, 64, 16, 64, torch.device("cpu"), torch.float32, kv_format="mxfp8")
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        fsi.decode_attention(torch.randn(1, 2, 64), c, pos=0, window=4, remote_pages=None, remote_counts=None, scale=1.0)
