"""Attention of a prompt over a sliding window and the first tokens ("sinks"), with gradients.

The single-token form over a paged cache is attention.decode_attention(..., sinks=n).  The
reference has no counterpart: its local window is always joined by whole routed pages
(foveal_indexer/attention.py:148-178).
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
import torch.nn.functional as F
from torch import Tensor

from . import _lib

_WHAT = "sink_window_attention"
_MFMA_WIDTHS = (64, 128, 256)  # head_dims of the bf16 MFMA kernels
# Products (queries x keys x head_dim) from which bf16 heads of other sizes are padded with zeros to
# the next of them: the copies cost 30-40 us of host time, 90 with gradients.  8 heads of 96 over
# 1024 tokens, window 512 (4e8): 291 us with gradients on fp32 MFMA, 275 padded; 40 (2e8): 203 and
# 269; 200 (8e8): 849 and 283; 2 x 4096 tokens, 32 heads of 96: 5247 and 811.
_PAD_WORK = 1 << 29


def _width(q: Tensor, keys: int) -> int:
    """head_dim to run q at."""
    hd = q.shape[3]
    if q.dtype != torch.bfloat16 or hd in _MFMA_WIDTHS or q.numel() * keys < _PAD_WORK:
        return hd
    return next((w for w in _MFMA_WIDTHS if w > hd), hd)


def _rows(t: Tensor) -> Tensor:
    """t with unit stride over head_dim; the other strides are the kernels' to follow.  bf16 rows that
    the bf16 MFMA kernels cannot read in 16-byte pieces are copied."""
    if t.stride(3) != 1:
        return t.contiguous()
    if (t.dtype == torch.bfloat16 and t.shape[3] in _MFMA_WIDTHS
            and (t.data_ptr() % 16 or any(s % 8 for s in t.stride()[:3]))):
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _out_like(q: Tensor) -> Tensor:
    """A (B, Hq, Tq, hd) view of a (B, Tq, Hq, hd) buffer: the heads merge without a copy."""
    B, Hq, Tq, hd = q.shape
    return q.new_empty((B, Tq, Hq, hd)).transpose(1, 2)


def _fwd_fake(q, k, v, lengths, window, sinks, scale, grad):
    lo = _out_like(q) if grad and q.dtype == torch.bfloat16 else q.new_empty((0,))
    return _out_like(q), q.new_empty(q.shape[:3] if grad else (0,), dtype=torch.float32), lo


@_lib.fsi_op("sink_window_attention", _fwd_fake)
def _fwd_op(q: Tensor, k: Tensor, v: Tensor, lengths: Optional[Tensor], window: int, sinks: int, scale: float,
            grad: bool) -> Tuple[Tensor, Tensor, Tensor]:
    """fsi_sink_attn: (out (B, Hq, Tq, hd), and for the backward lse (B, Hq, Tq) and, bf16, out's
    rounding remainder; else empty)."""
    dev = q.device
    q, k, v = _rows(q), _rows(k), _rows(v)
    B, Hq, Tq, hd = q.shape
    out = _out_like(q)
    lse = torch.empty((B, Hq, Tq) if grad else (0,), dtype=torch.float32, device=dev)
    lo = _out_like(q) if grad and q.dtype == torch.bfloat16 else q.new_empty((0,))
    L = _lib.lib()
    Hkv, Tk = k.shape[1], k.shape[2]
    need = L.fsi_sink_attn_workspace_size(B, Hq, Hkv, Tq, Tk, hd, window, sinks)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    with _lib.device_guard(dev):
        st = L.fsi_sink_attn(
            q.data_ptr(), *q.stride()[:3], k.data_ptr(), *k.stride()[:3], v.data_ptr(), *v.stride()[:3], B, Hq, Hkv,
            Tq, Tk, hd, window, sinks, _lib.ptr(lengths), scale, _lib.dtype_code(q.dtype, _WHAT), out.data_ptr(),
            *out.stride()[:3], lo.data_ptr() if lo.numel() else None, lse.data_ptr() if grad else None, _lib.ptr(ws),
            need, _lib.stream_handle(dev))
    _lib.check(st, _WHAT)
    return out, lse, lo


def _bwd_fake(q, k, v, out, lo, dout, lse, lengths, window, sinks, scale):
    return tuple(torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v))


@_lib.fsi_op("sink_window_attention_bwd", _bwd_fake)
def _bwd_op(q: Tensor, k: Tensor, v: Tensor, out: Tensor, lo: Tensor, dout: Tensor, lse: Tensor,
            lengths: Optional[Tensor], window: int, sinks: int, scale: float) -> Tuple[Tensor, Tensor, Tensor]:
    """fsi_sink_attn_bwd: contiguous (dq, dk, dv) of the operands' dtype."""
    dev = q.device
    q, k, v, dout = (_rows(t) for t in (q, k, v, dout))
    if out.stride(3) != 1 or (lo.numel() and lo.stride() != out.stride()):  # the kernels read both by out's strides
        out, lo = out.contiguous(), lo.contiguous()
    B, Hq, Tq, hd = q.shape
    Hkv, Tk = k.shape[1], k.shape[2]
    dq, dk, dv = (torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v))
    L = _lib.lib()
    need = L.fsi_sink_attn_bwd_workspace_size(B, Hq, Hkv, Tq, Tk, hd, window, sinks)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    with _lib.device_guard(dev):
        st = L.fsi_sink_attn_bwd(
            q.data_ptr(), *q.stride()[:3], k.data_ptr(), *k.stride()[:3], v.data_ptr(), *v.stride()[:3],
            out.data_ptr(), *out.stride()[:3], lo.data_ptr() if lo.numel() else None, dout.data_ptr(),
            *dout.stride()[:3], lse.data_ptr(), B, Hq, Hkv, Tq, Tk, hd, window, sinks, _lib.ptr(lengths), scale,
            _lib.dtype_code(q.dtype, _WHAT), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _lib.ptr(ws), need,
            _lib.stream_handle(dev))
    _lib.check(st, f"{_WHAT} backward")
    return dq, dk, dv


class _SinkAttnFn(torch.autograd.Function):
    """sink_window_attention with gradients for q, k and v: the forward keeps each row's softmax
    denominator and (bf16) what rounding took from its output, and the backward forms P again tile by
    tile."""

    @staticmethod
    def forward(ctx, q, k, v, lengths, window, sinks, scale):
        out, lse, lo = _fwd_op(q, k, v, lengths, window, sinks, scale, True)
        ctx.save_for_backward(q, k, v, out, lo, lse, lengths)
        ctx.meta = (window, sinks, scale)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lo, lse, lengths = ctx.saved_tensors
        grads = _bwd_op(q, k, v, out, lo, dout.to(q.dtype), lse, lengths, *ctx.meta)
        return (*grads, None, None, None, None)


def sink_window_attention(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    *,
    window: int,
    sinks: int = 0,
    scale: Optional[float] = None,
    lengths: Optional[Tensor] = None,
) -> Tensor:
    """Causal attention of q (B, Hq, Tq, hd) over k, v (B, Hkv, Tk, hd), Tq <= Tk, in which query
    i at position p = i + Tk - Tq sees the last `window` tokens up to itself and the first
    `sinks` tokens: keys s <= p with s > p - window or s < sinks.

    lengths: (B,) integers, tokens of each padded sequence.  Queries and keys at positions
    from a sequence's length on take no part: their output and gradients are 0, and their
    memory may hold anything.  A query that sees no key (window 0 without sinks) gets 0.
    bf16 or fp32, hd up to 256, softmax and sums in fp32; views with unit stride over hd are
    read in place.  scale defaults to 1 / sqrt(hd).  Differentiable (once) in q, k and v.
    Inside a length, v where it is hidden enters as 0 times the value, in the gradients q, k
    and the incoming gradient as well, so they have to be finite; hidden k may hold anything
    in the forward.  Returns (B, Hq, Tq, hd), a view of a
    (B, Tq, Hq, hd) buffer (of padded heads where hd is not a size of the MFMA kernels)."""
    dev = _lib.require_gpu(q, k, v, lengths, what=_WHAT)
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError(f"{_WHAT}: q, k, v dtypes {q.dtype}, {k.dtype}, {v.dtype} differ")
    _lib.dtype_code(q.dtype, _WHAT)
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape:
        raise ValueError(f"{_WHAT}: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} do not match")
    B, Hq, Tq, hd = q.shape
    Hkv, Tk = k.shape[1], k.shape[2]
    if k.shape[0] != B or k.shape[3] != hd or Hkv == 0 or Hq % Hkv or Tq > Tk:
        raise ValueError(f"{_WHAT}: q {tuple(q.shape)} and k {tuple(k.shape)} do not match "
                         "(one batch and head_dim, Hq a multiple of Hkv, Tq <= Tk)")
    if window < 0 or sinks < 0:
        raise ValueError(f"{_WHAT}: window {window} and sinks {sinks} must not be negative")
    if scale is None:
        scale = 1.0 / math.sqrt(hd)
    if lengths is not None:
        if lengths.is_floating_point() or lengths.numel() != B:
            raise ValueError(f"{_WHAT}: lengths must be {B} integers, got {tuple(lengths.shape)} {lengths.dtype}")
        lengths = lengths.to(device=dev, dtype=torch.int32).reshape(-1).contiguous()
    args = (lengths, int(window), int(sinks), float(scale))
    width = _width(q, min(Tk, window + sinks))
    if width != hd:
        q, k, v = (F.pad(t, (0, width - hd)) for t in (q, k, v))
        return _attend(q, k, v, args)[..., :hd]
    return _attend(q, k, v, args)


def _attend(q: Tensor, k: Tensor, v: Tensor, args) -> Tensor:
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _SinkAttnFn.apply(q, k, v, *args)
    return _fwd_op(q.detach(), k.detach(), v.detach(), *args, False)[0]
