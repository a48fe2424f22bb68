"""Measured calls of the quantised K/V cache and of windowed attention with sinks.

Three kinds of case:
  cache   a prompt (or one token) written into a cache held in 4 or 8 bits and read back
          (FovealKVCache(kv_format=...).load_dense, to_dense);
  decode  one query token per sequence over a cache in 4 bits, 8 bits or bf16: sinks, window
          and listed pages (decode_attention);
  sink    attention of a prompt over a sliding window and the first tokens, forward alone or
          with its gradients (sink_window_attention).

`own` chooses between the package's calls and the plain torch form of the same operators;
`exact` is the definition in 64 bits, written apart from the plain form.
"""
import math

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
DTYPES = {"bf16": BF16, "fp32": F32}
ELEM = {"bf16": 2, "fp32": 4}
PAGE = 64
GROUP = 32  # dims that share a scale
# bytes an element takes in the cache, its share of the scale byte included
CACHE_BYTES = {"mxfp4": 0.5 + 1 / GROUP, "mxfp8": 1 + 1 / GROUP, "bf16": 2.0}


def _package():
    from __graft_entry__ import load_package

    return load_package()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def listed():
    return [
        # the first token of a small batch: one append and its read back, latency only
        dict(name="cache4_token", kind="cache", fmt="mxfp4", dtype="bf16", B=16, Hkv=8, hd=128, start=0, n=1),
        # prompts of four sequences of the benchmark's 8B-class layer
        dict(name="cache4_prompt", kind="cache", fmt="mxfp4", dtype="bf16", B=4, Hkv=8, hd=128, start=0, n=8192),
        # fp32 model, odd heads and head size, a prompt that continues inside a page
        dict(name="cache8_odd", kind="cache", fmt="mxfp8", dtype="fp32", B=3, Hkv=5, hd=96, start=37, n=1003),
        # one sequence just past two pages: latency
        dict(name="decode4_short", kind="decode", fmt="mxfp4", dtype="bf16", B=1, Hq=8, Hkv=2, hd=64, ctx=130,
             window=1 << 20, sinks=0, pages=0, ragged=False),
        # the foveal decode step of the benchmark (local window and 32 routed pages), 32768 tokens cached
        dict(name="decode4_foveal", kind="decode", fmt="mxfp4", dtype="bf16", B=32, Hq=32, Hkv=8, hd=128, ctx=32768,
             window=1024, sinks=0, pages=32, ragged=False),
        # every token of a long context attended
        dict(name="decode4_full", kind="decode", fmt="mxfp4", dtype="bf16", B=8, Hq=32, Hkv=8, hd=128, ctx=65536,
             window=1 << 20, sinks=0, pages=0, ragged=False),
        # sequences of different lengths, window and sinks, 8 bits, 8 query heads per KV head
        dict(name="decode8_sinks", kind="decode", fmt="mxfp8", dtype="bf16", B=48, Hq=16, Hkv=2, hd=64, ctx=9001,
             window=4096, sinks=4, pages=0, ragged=True),
        # fp32 model, three query heads per KV head, odd sizes
        dict(name="decode4_fp32", kind="decode", fmt="mxfp4", dtype="fp32", B=3, Hq=15, Hkv=5, hd=96, ctx=2500,
             window=700, sinks=5, pages=7, ragged=True),
        # window and sinks over the bf16 pages that the framework has held all along
        dict(name="decode16_sinks", kind="decode", fmt="bf16", dtype="bf16", B=64, Hq=32, Hkv=8, hd=128, ctx=8192,
             window=1024, sinks=4, pages=0, ragged=True),
        # a long prompt, forward only
        dict(name="sink_prompt", kind="sink", dtype="bf16", B=1, Hq=32, Hkv=8, hd=128, Tq=16384, Tk=16384,
             window=4096, sinks=4, lengths=False, grad=False),
        # a training step's attention
        dict(name="sink_train", kind="sink", dtype="bf16", B=2, Hq=32, Hkv=8, hd=128, Tq=4096, Tk=4096, window=1024,
             sinks=4, lengths=False, grad=True),
        # a padded fp32 batch of odd lengths with its gradients
        dict(name="sink_train_fp32", kind="sink", dtype="fp32", B=3, Hq=6, Hkv=3, hd=64, Tq=333, Tk=333, window=100,
             sinks=3, lengths=True, grad=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["cache", "decode", "decode", "sink", "sink"])
    if kind == "cache":
        fmt, dtype = rng.choice(["mxfp4", "mxfp8"]), rng.choice(["bf16", "fp32"])
        B, Hkv, hd = rng.randint(1, 16), rng.randint(1, 8), rng.choice([64, 96, 128, 256])
        n = min(_log_int(rng, 1, 8192), max(1, (1 << 25) // (B * Hkv * hd)))
        return dict(kind=kind, fmt=fmt, dtype=dtype, B=B, Hkv=Hkv, hd=hd, start=rng.choice([0, rng.randint(0, 200)]),
                    n=n)
    if kind == "decode":
        fmt = rng.choice(["mxfp4", "mxfp4", "mxfp8", "bf16"])
        dtype = "bf16" if fmt == "bf16" else rng.choice(["bf16", "bf16", "fp32"])
        Hkv, hd = rng.randint(1, 8), rng.choice([64, 128] if fmt == "bf16" else [64, 96, 128, 256])
        Hq, B = Hkv * rng.choice([1, 2, 3, 4, 7, 8, 16]), _log_int(rng, 1, 64)
        ctx = min(_log_int(rng, 1, 65536), max(64, (1 << 28) // (B * Hkv * hd)))
        # the bf16 pages without sinks are an older path, with results of its own
        sinks = rng.randint(1, 70) if fmt == "bf16" else rng.choice([0, rng.randint(1, 70)])
        window = rng.choice([1 << 20, _log_int(rng, 1, 4096), _log_int(rng, 1, 4096)])
        pages = rng.choice([0, rng.randint(1, 40)])
        return dict(kind=kind, fmt=fmt, dtype=dtype, B=B, Hq=Hq, Hkv=Hkv, hd=hd, ctx=ctx, window=window, sinks=sinks,
                    pages=pages, ragged=rng.random() < 0.7)
    dtype, grad = rng.choice(["bf16", "bf16", "fp32"]), rng.random() < 0.7
    hd = rng.choice([32, 64, 64, 80, 96, 128, 128])
    Hkv = rng.randint(1, 8)
    Hq, B = Hkv * rng.choice([1, 2, 3, 4, 8]), rng.randint(1, 4)
    # no more multiplications than the listed case of its type
    pairs = (1 << 29 if dtype == "bf16" and hd in (64, 128) else 1 << 25) // (B * Hq)
    Tk = min(_log_int(rng, 1, 8192), max(16, int(math.sqrt(2 * pairs))))
    window = rng.choice([Tk, min(Tk, _log_int(rng, 1, 4096)), min(Tk, _log_int(rng, 1, 4096))])
    Tq = rng.choice([Tk, Tk, rng.randint(1, Tk)])
    return dict(kind=kind, dtype=dtype, B=B, Hq=Hq, Hkv=Hkv, hd=hd, Tq=Tq, Tk=Tk, window=window,
                sinks=rng.choice([0, 4, rng.randint(1, 70)]), lengths=rng.random() < 0.4, grad=grad)


# --- inputs ------------------------------------------------------------------------------


def _channels(c, g):
    """Per-channel standard deviations of K: a few channels of a head are far larger."""
    return torch.randn(c["Hkv"], 1, c["hd"], device="cuda", generator=g).mul_(0.8).exp_()


def _kv_chunks(c, seed, n, step=4096):
    """(first token, K, V) of tokens [0, n) in pieces, (B, Hkv, piece, hd) of the case's type."""
    g, dt = _gen(seed), DTYPES[c["dtype"]]
    kstd = _channels(c, g)
    for t in range(0, n, step):
        shape = (c["B"], c["Hkv"], min(step, n - t), c["hd"])
        k = torch.randn(shape, device="cuda", generator=g).mul_(kstd).to(dt)
        v = torch.randn(shape, device="cuda", generator=g).to(dt)
        yield t, k, v


def _positions(c):
    """Position of each sequence's query token: the context's last, or spread over its second half."""
    B, ctx = c["B"], c["ctx"]
    return [ctx - 1 - (b * ctx) // (2 * B) if c["ragged"] else ctx - 1 for b in range(B)]


def _first_local(c, pos):
    return max(0, pos + 1 - c["window"])


def _page_counts(c):
    return [min(c["pages"], _first_local(c, p) // PAGE) for p in _positions(c)]


def _decode_inputs(c, seed):
    g = _gen(seed + 1)
    q = torch.randn(c["B"], c["Hq"], c["hd"], device="cuda", generator=g).to(DTYPES[c["dtype"]])
    pages = None
    if c["pages"]:
        pages = torch.full((c["B"], c["pages"]), -1, dtype=torch.int32, device="cuda")
        for b, (p, cnt) in enumerate(zip(_positions(c), _page_counts(c))):
            if cnt:
                perm = torch.randperm(_first_local(c, p) // PAGE, device="cuda", generator=g)
                pages[b, :cnt] = perm[:cnt].to(torch.int32)
    n_pages = -(-c["ctx"] // PAGE)
    table = torch.randperm(c["B"] * n_pages, device="cuda", generator=g).to(torch.int32).view(c["B"], n_pages)
    return q, pages, table


def _sink_inputs(c, seed):
    g, dt = _gen(seed), DTYPES[c["dtype"]]

    def heads(T, H):  # (B, H, T, hd) views of a projection's (B, T, H hd) output
        return torch.randn(c["B"], T, H, c["hd"], device="cuda", generator=g).to(dt).transpose(1, 2)

    q, k, v, dout = heads(c["Tq"], c["Hq"]), heads(c["Tk"], c["Hkv"]), heads(c["Tk"], c["Hkv"]), heads(c["Tq"], c["Hq"])
    lengths = None
    if c["lengths"]:
        lengths = torch.randint(max(1, c["Tk"] // 2), c["Tk"] + 1, (c["B"],), device="cuda", generator=g)
        lengths = lengths.to(torch.int32)
    return q, k, v, dout, lengths


# --- the plain form -------------------------------------------------------------------------


def _pow2(e):
    """2^e for integer tensors e in [-126, 127], exactly."""
    return ((e.to(torch.int32) + 127) << 23).view(F32)


def _plain_quantise(x, fmt):
    """(element values, e) of x (..., hd): element * 2^e per group of 32 dims."""
    x = x.float().unflatten(-1, (-1, GROUP))
    mant, ex = torch.frexp(x.abs().amax(-1, keepdim=True))  # mant in [0.5, 1)
    top, limit = (2, 0.875) if fmt == "mxfp4" else (8, 0.90625)
    e = ex - 1 - top + (mant > limit).to(ex.dtype)
    e = torch.where(mant == 0, torch.full_like(e, -116), e).clamp(-116, 127 - top)
    y = x * _pow2(-e)
    _, ey = torch.frexp(y)
    low, bits = (0, 1) if fmt == "mxfp4" else (-6, 3)
    shift = (ey - 1).clamp(min=low) - bits
    y = torch.round(y * _pow2(-shift)) * _pow2(shift)
    peak = 6.0 if fmt == "mxfp4" else 448.0
    return y.clamp(-peak, peak), e


def _plain_dequantise(y, e):
    return (y * _pow2(e)).flatten(-2)


_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _plain_store(x, fmt):
    """The plain form's cache of x: packed element codes and scale bytes."""
    y, e = _plain_quantise(x, fmt)
    y, scale = y.flatten(-2), (e.squeeze(-1) + 127).to(torch.uint8)
    if fmt == "mxfp8":
        return y.to(torch.float8_e4m3fn).view(torch.uint8), scale
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=x.device)
    code = torch.bucketize(y.abs(), mids).to(torch.uint8) | (torch.signbit(y).to(torch.uint8) << 3)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def _plain_load(codes, scale, fmt):
    if fmt == "mxfp8":
        y = codes.view(torch.float8_e4m3fn).float()
    else:
        lut = torch.tensor(_E2M1 + [-t for t in _E2M1], device=codes.device)
        y = torch.stack((lut[(codes & 15).long()], lut[(codes >> 4).long()]), -1).flatten(-2)
    return _plain_dequantise(y.unflatten(-1, (-1, GROUP)), scale.unsqueeze(-1).to(torch.int32) - 127)


def _plain_cache(s):
    c, outs = s["case"], []
    for x in (s["k"], s["v"]):
        full = torch.zeros(c["B"], c["Hkv"], c["start"] + c["n"], c["hd"], dtype=x.dtype, device=x.device)
        full[:, :, c["start"]:] = _plain_dequantise(*_plain_quantise(x, c["fmt"])).to(x.dtype)
        outs.append(full)
    return outs


def _plain_tokens(c, pos, pages, counts):
    """Token of every support slot (B, S) and whether it is attended."""
    dev = pos.device
    ls = (pos + 1 - c["window"]).clamp(min=0)
    sink_end = ls.clamp(max=c["sinks"])
    sink = torch.arange(c["sinks"], device=dev).expand(c["B"], -1)
    win = ls[:, None] + torch.arange(min(c["window"], c["ctx"]), device=dev)
    toks, ok = [sink, win], [sink < sink_end[:, None], win <= pos[:, None]]
    if pages is not None:
        t = pages.long()[:, :, None] * PAGE + torch.arange(PAGE, device=dev)
        live = torch.arange(c["pages"], device=dev)[None, :, None] < counts[:, None, None]
        toks.append(t.flatten(1))
        ok.append((live & (t >= sink_end[:, None, None]) & (t < ls[:, None, None])).flatten(1))
    toks, ok = torch.cat(toks, 1), torch.cat(ok, 1)
    return torch.where(ok, toks, 0), ok


def _plain_decode(s):
    c = s["case"]
    toks, ok = _plain_tokens(c, s["pos"].long(), s["pages"], s["counts"])

    def gather(cache):
        parts = [x.gather(2, toks[:, None, :, None].expand(-1, c["Hkv"], -1, x.shape[-1])) for x in cache]
        return _plain_load(*parts, c["fmt"]) if len(parts) == 2 else parts[0].float()

    q = s["q"].float().view(c["B"], c["Hkv"], -1, c["hd"])
    x = torch.matmul(q, gather(s["k"]).transpose(-1, -2).contiguous()) / math.sqrt(c["hd"])
    x = x.masked_fill(~ok[:, None, None], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    o = torch.matmul(p, gather(s["v"])) / p.sum(-1, keepdim=True)
    return o.view(c["B"], c["Hq"], c["hd"]).to(s["q"].dtype)


def _plain_sink_forward(c, q, k, v, lengths):
    """fp32 attention in blocks of queries against their window and the sinks."""
    B, Hkv, G, hd = c["B"], c["Hkv"], c["Hq"] // c["Hkv"], c["hd"]
    Tq, Tk, W, off = c["Tq"], c["Tk"], c["window"], c["Tk"] - c["Tq"]
    dev, outs, step = q.device, [], 512
    for i in range(0, Tq, step):
        n = min(step, Tq - i)
        lo, hi = max(0, off + i - W + 1), off + i + n
        keys = torch.cat((torch.arange(min(c["sinks"], lo), device=dev), torch.arange(lo, hi, device=dev)))
        p = torch.arange(off + i, hi, device=dev)
        ok = (keys <= p[:, None]) & ((keys > p[:, None] - W) | (keys < c["sinks"]))
        ok = ok.expand(B, 1, 1, n, -1)
        if lengths is not None:
            n_b = lengths.view(B, 1, 1, 1, 1)
            ok = ok & (keys < n_b) & (p[:, None] < n_b)
        x = torch.matmul(q[:, :, i:i + n].reshape(B, Hkv, G * n, hd),
                         k[:, :, keys].transpose(-1, -2).contiguous()) / math.sqrt(hd)
        x = x.view(B, Hkv, G, n, -1).masked_fill(~ok, -math.inf)
        top = x.amax(-1, keepdim=True)
        e = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
        e = e / e.sum(-1, keepdim=True).clamp(min=1e-30)
        outs.append(torch.matmul(e.view(B, Hkv, G * n, -1), v[:, :, keys]).view(B, c["Hq"], n, hd))
    return torch.cat(outs, 2)


def _plain_sink(s):
    c, (q, k, v, dout, lengths) = s["case"], s["tensors"]
    qf, kf, vf = (t.detach().float().requires_grad_(c["grad"]) for t in (q, k, v))
    out = _plain_sink_forward(c, qf, kf, vf, lengths)
    if not c["grad"]:
        return out.to(q.dtype)
    grads = torch.autograd.grad(out, (qf, kf, vf), dout.float())
    return (out.detach().to(q.dtype), *(t.to(q.dtype) for t in grads))


# --- the measured call ------------------------------------------------------------------------


def _cache_of(c, n, table=None):
    fmt = None if c["fmt"] == "bf16" else c["fmt"]
    return _package().FovealKVCache(c["B"], n, c["Hkv"], c["hd"], 16, PAGE, torch.device("cuda"), DTYPES[c["dtype"]],
                                    page_table=table, kv_format=fmt)


def prepare(case, seed):
    c, s = dict(case), {"case": dict(case)}
    if c["kind"] == "cache":
        _, s["k"], s["v"] = next(_kv_chunks(c, seed, c["n"], step=c["n"]))
        if own:
            s["cache"] = _cache_of(c, c["start"] + c["n"])
        return s
    if c["kind"] == "sink":
        s["tensors"] = _sink_inputs(c, seed)
        if own and c["grad"]:
            s["tensors"] = tuple(t.requires_grad_() for t in s["tensors"][:3]) + s["tensors"][3:]
        return s
    s["q"], s["pages"], table = _decode_inputs(c, seed)
    s["pos"] = torch.tensor(_positions(c), dtype=torch.int32, device="cuda")
    s["counts"] = torch.tensor(_page_counts(c), dtype=torch.int32, device="cuda")
    if own:
        s["cache"] = _cache_of(c, c["ctx"], table)
        for t, k, v in _kv_chunks(c, seed, c["ctx"]):
            s["cache"].load_dense(k, v, start=t)
        return s
    ks, vs = [], []
    for _, k, v in _kv_chunks(c, seed, c["ctx"]):
        ks.append((k,) if c["fmt"] == "bf16" else _plain_store(k, c["fmt"]))
        vs.append((v,) if c["fmt"] == "bf16" else _plain_store(v, c["fmt"]))
    s["k"], s["v"] = (tuple(torch.cat(parts, 2) for parts in zip(*x)) for x in (ks, vs))
    return s


def run(state):
    c = state["case"]
    if c["kind"] == "cache":
        if not own:
            return _plain_cache(state)
        state["cache"].load_dense(state["k"], state["v"], start=c["start"])
        return state["cache"].to_dense(c["start"] + c["n"])
    if c["kind"] == "decode":
        if not own:
            return _plain_decode(state)
        return _package().decode_attention(
            state["q"], state["cache"], pos=state["pos"], window=c["window"], remote_pages=state["pages"],
            remote_counts=state["counts"], scale=1.0 / math.sqrt(c["hd"]), sinks=c["sinks"])
    if not own:
        return _plain_sink(state)
    q, k, v, dout, lengths = state["tensors"]
    out = _package().sink_window_attention(q, k, v, window=c["window"], sinks=c["sinks"], lengths=lengths)
    if not c["grad"]:
        return out
    return (out.detach(), *torch.autograd.grad(out, (q, k, v), dout))


def _support(c):
    """Attended tokens of every sequence of a decode case, summed."""
    total = 0
    for p, cnt in zip(_positions(c), _page_counts(c)):
        ls = _first_local(c, p)
        # pages are drawn at random: those that hold sinks are few enough to leave out of the count
        total += min(c["sinks"], ls) + p + 1 - ls + PAGE * cnt
    return total


def work(case):
    c = case
    if c["kind"] == "cache":
        n = 2 * c["B"] * c["Hkv"] * c["n"] * c["hd"]
        back = 2 * c["B"] * c["Hkv"] * (c["start"] + c["n"]) * c["hd"]
        b = ELEM[c["dtype"]]
        return {"bytes": int(n * (b + CACHE_BYTES[c["fmt"]]) + back * (b + CACHE_BYTES[c["fmt"]])), "flops": 2 * n}
    if c["kind"] == "decode":
        n = _support(c)
        io = 2 * c["B"] * c["Hq"] * c["hd"] * ELEM[c["dtype"]]
        return {"bytes": int(2 * n * c["Hkv"] * c["hd"] * CACHE_BYTES[c["fmt"]]) + io,
                "flops": 4 * n * c["Hq"] * c["hd"]}
    p = torch.arange(c["Tk"] - c["Tq"], c["Tk"], dtype=torch.int64)
    pairs = int(((p + 1).clamp(max=c["window"]) + (p + 1 - c["window"]).clamp(min=0, max=c["sinks"])).sum())
    b = ELEM[c["dtype"]]
    io = c["B"] * c["hd"] * b * (2 * c["Hq"] * c["Tq"] + 2 * c["Hkv"] * c["Tk"])
    return {"bytes": io * (2 if c["grad"] else 1),
            "flops": (14 if c["grad"] else 4) * pairs * c["B"] * c["Hq"] * c["hd"]}


# --- the definition in 64 bits ------------------------------------------------------------------


def _exact_grid(fmt):
    """The element values >= 0 in ascending order: exponent field, then mantissa field."""
    ebits, mbits, bias = (2, 1, 1) if fmt == "mxfp4" else (4, 3, 7)
    vals = []
    for ef in range(1 << ebits):
        for mf in range(1 << mbits):
            frac = mf / (1 << mbits)
            vals.append(frac * 2.0 ** (1 - bias) if ef == 0 else (1 + frac) * 2.0 ** (ef - bias))
    return vals if fmt == "mxfp4" else vals[:-1]  # the last e4m3 pattern is NaN


def _exact_cache_values(x, fmt):
    """What the cache holds for x (..., hd), in 64 bits."""
    grid = torch.tensor(_exact_grid(fmt), dtype=F64, device=x.device)
    limit = float(grid[-1] + (grid[-1] - grid[-2]) / 2)  # half a step above the largest element
    x = x.to(F64).unflatten(-1, (-1, GROUP))
    a = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(a.clamp(min=1e-300) / limit)).clamp(-400, 400)
    for shift in (1, 0, -1):  # the smallest e with a <= limit 2^e, whatever log2 rounded to
        e = torch.where(a <= limit * torch.exp2(e - 1), e - 1, torch.where(a > limit * torch.exp2(e), e + 1, e))
    e = e.clamp(-116, 127 - math.floor(math.log2(float(grid[-1]))))
    y = x.abs() / torch.exp2(e)
    mids = (grid[1:] + grid[:-1]) / 2
    i = torch.bucketize(y.contiguous(), mids)  # number of midpoints below y
    tie = (i < len(mids)) & (y == mids[i.clamp(max=len(mids) - 1)]) & (i % 2 == 1)
    return (torch.sign(x) * grid[i + tie.long()] * torch.exp2(e)).flatten(-2)


def _exact_cache(c, seed):
    outs = []
    _, k, v = next(_kv_chunks(c, seed, c["n"], step=c["n"]))
    for x in (k, v):
        held = torch.cat([_exact_cache_values(t, c["fmt"]) for t in x.split(1)])
        outs.append(torch.nn.functional.pad(held, (0, 0, c["start"], 0)))
    return outs


def _exact_decode(c, seed):
    q, pages, _ = _decode_inputs(c, seed)
    toks = []
    for b, (p, cnt) in enumerate(zip(_positions(c), _page_counts(c))):
        seen = set(range(_first_local(c, p), p + 1)) | set(range(min(c["sinks"], p + 1)))
        for pg in (pages[b, :cnt].tolist() if cnt else []):
            seen |= set(range(pg * PAGE, pg * PAGE + PAGE))
        toks.append(torch.tensor(sorted(seen), device="cuda"))
    kept_k, kept_v = [[] for _ in toks], [[] for _ in toks]
    for t0, k, v in _kv_chunks(c, seed, c["ctx"]):
        for b, t in enumerate(toks):
            here = t[(t >= t0) & (t < t0 + k.shape[2])] - t0
            kept_k[b].append(k[b, :, here])
            kept_v[b].append(v[b, :, here])
    out = torch.empty(c["B"], c["Hq"], c["hd"], dtype=F64, device="cuda")
    for b in range(c["B"]):
        k, v = torch.cat(kept_k[b], 1), torch.cat(kept_v[b], 1)
        if c["fmt"] != "bf16":
            k, v = _exact_cache_values(k, c["fmt"]), _exact_cache_values(v, c["fmt"])
        k, v = k.to(F64), v.to(F64)
        qb = q[b].to(F64).view(c["Hkv"], -1, c["hd"])
        p = torch.softmax(torch.matmul(qb, k.transpose(1, 2).contiguous()) / math.sqrt(c["hd"]), -1)
        out[b] = torch.matmul(p, v).view(c["Hq"], c["hd"])
    return out


def _exact_sink(c, seed):
    q, k, v, dout, lengths = _sink_inputs(c, seed)
    G, off, scale, W = c["Hq"] // c["Hkv"], c["Tk"] - c["Tq"], 1.0 / math.sqrt(c["hd"]), c["window"]
    out = torch.zeros(q.shape, dtype=F64, device=q.device)
    dq, dk, dv = torch.zeros_like(out), *(torch.zeros(k.shape, dtype=F64, device=k.device) for _ in range(2))
    step = 1024
    for b in range(c["B"]):
        n_b = int(lengths[b]) if lengths is not None else c["Tk"]
        for h in range(c["Hq"]):
            qh, gh = q[b, h].to(F64), dout[b, h].to(F64)
            kh, vh = k[b, h // G].to(F64), v[b, h // G].to(F64)
            for i in range(0, max(0, n_b - off), step):
                j = min(i + step, n_b - off)
                # every key of the block's windows, and before them the sinks (or all keys up to there)
                lo, hi = max(0, off + i + 1 - W), off + j
                sel = torch.tensor(list(range(min(c["sinks"], lo))) + list(range(lo, hi)), device=q.device)
                rows = torch.arange(off + i, off + j, device=q.device)[:, None]
                hidden = (sel > rows) | ((sel <= rows - W) & (sel >= c["sinks"]))
                p = torch.softmax((qh[i:j] @ kh[sel].T * scale).masked_fill(hidden, -math.inf), -1)
                o = p @ vh[sel]
                out[b, h, i:j] = o
                if c["grad"]:
                    ds = p * (gh[i:j] @ vh[sel].T - (gh[i:j] * o).sum(-1, keepdim=True)) * scale
                    dq[b, h, i:j] = ds @ kh[sel]
                    dk[b, h // G].index_add_(0, sel, ds.T @ qh[i:j])
                    dv[b, h // G].index_add_(0, sel, p.T @ gh[i:j])
    return (out, dq, dk, dv) if c["grad"] else out


def exact(case, seed):
    return {"cache": _exact_cache, "decode": _exact_decode, "sink": _exact_sink}[case["kind"]](dict(case), seed)
