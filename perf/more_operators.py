"""Serving in fewer bits, in its plain form and through the library: a paged KV cache held in 8 or 4 bits (quantised as it is written,
read back, attended to token by token), and linear layers in 8-bit integers.

`listed()` names the fixed cases, `draw()` gives more of the same ranges, `prepare()` builds what a program holds before the call,
`run()` is one call (`own` false: elementary torch operations in 32 bits; true: the library's operators), `work()` what it cannot do
without, `exact()` the results by the definition in 64 bits.

Kinds of case:
  cache    the new tokens of a batch are quantised into their places of the cache, then all keys and values of the batch are read back
  decode   one query token per sequence attends to the quantised keys and values: the last `window` (0: all) and the first `sinks`
  linear   rows of activations are quantised, one scale each, and multiplied by int8 weights with a scale per output channel

The cache's format. 8 bits: a row of D values of one token and head has one fp32 scale, value = (code - 128) scale, scale = max|x| / 127.
4 bits: every 64 values have a bf16 pair (step, least), value = least + step code; least is the minimum rounded down, step a fifteenth of what
lies above it, rounded up. Two codes per byte, the even index in the low half. Scales lie as [pages, heads, page], pairs as
[pages, heads, page, D / 64, 2].
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
HEADS = ((16, 16), (32, 8), (64, 8), (6, 1), (96, 12), (32, 2))
LEAST = 2.0 ** -100     # magnitudes below it count as it
MOST_FLOPS = 3.9e12     # about the largest listed case
MOST_BYTES = 2.5e9


def _cache(B, hkv, head_dim, new, kv, page, bits, dtype="bf16", ragged=False, fused=False):
    return dict(kind="cache", B=B, hkv=hkv, head_dim=head_dim, new=new, kv=kv, page=page, bits=bits, dtype=dtype, ragged=ragged, fused=fused)


def _decode(B, hq, hkv, head_dim, kv, page, bits, dtype="bf16", ragged=False, window=0, sinks=0, soft_cap=0.0):
    return dict(kind="decode", B=B, hq=hq, hkv=hkv, head_dim=head_dim, kv=kv, page=page, bits=bits, dtype=dtype, ragged=ragged,
                window=window, sinks=sinks, soft_cap=soft_cap)


def _linear(m, n, k, dtype="bf16"):
    return dict(kind="linear", m=m, n=n, k=k, dtype=dtype)


def listed():
    return [
        # one short request's first tokens: launch latency decides
        dict(name="cache8_small", **_cache(1, 8, 128, 17, 40, 16, 8)),
        # chunks of a few ragged prompts, k and v parts of a fused projection, 4 bits, an odd length
        dict(name="cache4_ragged", **_cache(5, 8, 128, 509, 3001, 16, 4, dtype="fp16", ragged=True, fused=True)),
        # 4096-token chunks of a few long prompts, read back for their attention
        dict(name="cache8_long", **_cache(4, 8, 128, 4096, 32768, 64, 8)),
        # one interactive request: launch latency decides
        dict(name="decode8_b1", **_decode(1, 32, 8, 128, 4096, 16, 8)),
        # a serving batch of all lengths
        dict(name="decode8_b32_ragged", **_decode(32, 32, 8, 128, 8192, 16, 8, ragged=True)),
        # one long document in 4 bits
        dict(name="decode4_b1_512k", **_decode(1, 32, 8, 128, 524288, 16, 4)),
        # a large batch of long conversations in 4 bits
        dict(name="decode4_b64_ragged", **_decode(64, 64, 8, 128, 16384, 64, 4, dtype="fp16", ragged=True)),
        # windowed layer with a soft cap, large heads of one kv head, odd sizes, pages of one token
        dict(name="decode8_b201_window", **_decode(201, 6, 1, 256, 2003, 1, 8, dtype="fp16", ragged=True, window=1024, sinks=4, soft_cap=30.0)),
        # a projection of one token: launch latency and the weights' bytes
        dict(name="linear_m1", **_linear(1, 4096, 4096)),
        # a decode step's batch on a large layer: the weights' bytes
        dict(name="linear_m16", **_linear(16, 6144, 12288)),
        # a short prompt, odd sizes
        dict(name="linear_m1000", **_linear(1000, 5504, 4096, dtype="fp16")),
        # a long prompt on a large layer: tensor rate
        dict(name="linear_m8192", **_linear(8192, 14336, 16384)),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread evenly over the logarithm."""
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("cache", "decode", "decode", "decode", "linear", "linear"))
    while True:
        hq, hkv = rng.choice(HEADS)
        head_dim, page = rng.choice((64, 128, 128, 256)), rng.choice((1, 16, 16, 64))
        bits, dtype = rng.choice((8, 4)), rng.choice(("bf16", "fp16"))
        if kind == "cache":
            new = _log(rng, 1, 8192)
            case = _cache(_log(rng, 1, 64), hkv, head_dim, new, _log(rng, new, 65536), page, bits, dtype, rng.random() < 0.5, rng.random() < 0.5)
        elif kind == "decode":
            windowed = rng.random() < 0.3
            case = _decode(_log(rng, 1, 256), hq, hkv, head_dim, _log(rng, 1, 524288), page, bits, dtype, rng.random() < 0.6,
                           _log(rng, 16, 8192) if windowed else 0, rng.choice((0, 4, 37)) if windowed else 0, rng.choice((0.0, 0.0, 30.0)))
        else:
            case = _linear(_log(rng, 1, 8192), 8 * _log(rng, 32, 4096), 16 * _log(rng, 16, 1024), dtype)
        if work(case)["flops"] <= MOST_FLOPS and _held(case) <= MOST_BYTES:
            return case


def _lens(case):
    """Keys per sequence, on the host. Ragged: evenly spread up to the largest."""
    B, kv = case["B"], case["kv"]
    return [max(1, kv * (i + 1) // B) if case["ragged"] else kv for i in range(B)]


def _news(case, lens):
    """New tokens of each sequence, the last ones of its keys."""
    return [min(n, max(1, case["new"] * n // case["kv"])) for n in lens]


def _row(case):
    """Bytes of one token and head, of k or of v, with its scales."""
    D = case["head_dim"]
    return D + 4 if case["bits"] == 8 else D // 2 + D // 16


def _held(case):
    """Bytes that a state and its outputs hold."""
    if case["kind"] == "linear":
        return 3.0 * case["m"] * case["k"] + 1.0 * case["n"] * case["k"] + 2.0 * case["m"] * case["n"]
    rows = 2.0 * case["B"] * case["hkv"] * (case["kv"] + case["page"])
    return rows * _row(case) + (rows * case["head_dim"] * 4 if case["kind"] == "cache" else 0.0)


def _seen(case, n):
    """Keys that a sequence's query sees."""
    w = case["window"]
    return n if w == 0 else min(n, w + min(case["sinks"], max(0, n - w)))


def work(case):
    if case["kind"] == "linear":
        m, n, k = 1.0 * case["m"], 1.0 * case["n"], 1.0 * case["k"]
        return {"bytes": 2 * m * k + n * k + 4 * n + 2 * m * n, "flops": 2 * m * n * k}
    lens, hkv, D = _lens(case), case["hkv"], case["head_dim"]
    if case["kind"] == "cache":
        new, keys = sum(_news(case, lens)), sum(lens)
        # new rows are read and written in fewer bits, all rows read in fewer bits and written
        return {"bytes": 2.0 * hkv * (new * (2 * D + _row(case)) + keys * (_row(case) + 2 * D)), "flops": 4.0 * hkv * D * (new + keys)}
    keys = sum(_seen(case, n) for n in lens)
    return {"bytes": 2.0 * keys * hkv * _row(case) + 4.0 * case["B"] * case["hq"] * D, "flops": 4.0 * keys * case["hq"] * D}


def _quotient(a, b):
    """a / b, rounded once (with a number on either side torch multiplies by a rounded reciprocal)."""
    t = a if isinstance(a, torch.Tensor) else b
    return torch.div(a if t is a else torch.full_like(t, a), b if t is b else torch.full_like(t, b))


def _bf16_down(x):
    """The largest bf16 that is not above x (fp32), as fp32."""
    b = x.to(torch.bfloat16)
    return torch.where(b.float() > x, torch.nextafter(b, torch.full_like(b, -math.inf)), b).float()


def _quantise(x, bits):
    """Rows [..., D] -> codes (one per byte, or two) and scales [...] / pairs [..., D / 64, 2]."""
    x = x.float()
    if bits == 8:
        most = x.abs().amax(-1, keepdim=True).clamp_min(LEAST)
        return (torch.round(x * _quotient(127.0, most)) + 128.0).to(torch.uint8), _quotient(most, 127.0).squeeze(-1)
    g = x.unflatten(-1, (-1, 64))
    least = _bf16_down(g.amin(-1, keepdim=True))
    step = -_bf16_down(-_quotient(g.amax(-1, keepdim=True) - least, 15.0).clamp_min(LEAST))
    code = torch.round((g - least) * _quotient(1.0, step)).clamp(0.0, 15.0).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.cat([step, least], -1).to(torch.bfloat16)


def _values(codes, scales, bits):
    """Codes and scales -> fp32 rows."""
    if bits == 8:
        return (codes.float() - 128.0) * scales.unsqueeze(-1)
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float().unflatten(-1, (-1, 64))
    p = scales.float()
    return (c * p[..., 0:1] + p[..., 1:2]).flatten(-2)


def _normal(gen, shape, dtype):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)


def _rows(gen, shape, dtype, channels):
    """Keys or values: normal, some channels (of all tokens) several times as large, as keys have them."""
    return _normal(gen, shape, dtype) * channels


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, s = DTYPES[case["dtype"]], {"case": dict(case)}
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        # activations: a few channels are ten times as large as the others
        channels = torch.where(torch.rand(k, generator=gen, device="cuda") < 0.01, 10.0, 1.0).to(dt)
        s["x"] = _normal(gen, (m, k), dt) * channels
        # weights, quantised when the model was loaded: a scale per output channel, the largest of each 127
        w = torch.empty((n, k), dtype=torch.int8, device="cuda")
        for n0 in range(0, n, 4096):
            part = _normal(gen, (min(4096, n - n0), k), torch.float32)
            w[n0:n0 + 4096] = torch.round(part * (127.0 / part.abs().amax(1, keepdim=True))).to(torch.int8)
        s["w"], s["w_scale"] = w, (0.5 + torch.rand(n, generator=gen, device="cuda")) * (4.0 / 127.0 * k ** -0.5)
        return s
    B, hkv, D, page, bits = case["B"], case["hkv"], case["head_dim"], case["page"], case["bits"]
    lens = _lens(case)
    random.Random(int(seed)).shuffle(lens)                      # lengths in no order
    per_seq = -(-max(lens) // page)
    pages = B * per_seq + 1
    width = D if bits == 8 else D // 2
    s["codes"] = torch.empty((2, pages, page, hkv, width), dtype=torch.uint8, device="cuda")
    s["scales"] = torch.empty((2, pages, hkv, page) + (() if bits == 8 else (D // 64, 2)), device="cuda",
                              dtype=torch.float32 if bits == 8 else torch.bfloat16)
    channels = torch.where(torch.rand((2, hkv, D), generator=gen, device="cuda") < 0.03, 6.0, 1.0).to(dt)
    step = max(1, (1 << 25) // (page * hkv * D))
    for i in range(2):
        for p0 in range(0, pages, step):
            codes, scales = _quantise(_rows(gen, (min(step, pages - p0), page, hkv, D), dt, channels[i]), bits)
            s["codes"][i, p0:p0 + step], s["scales"][i, p0:p0 + step] = codes, scales.transpose(1, 2)
    # pages as a running server hands them out: in no order
    s["table"] = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)[:B * per_seq].view(B, per_seq)
    s["host_lens"], s["lens"] = lens, torch.tensor(lens, dtype=torch.int32, device="cuda")
    if case["kind"] == "decode":
        s["q"], s["scale"] = _normal(gen, (B, case["hq"], D), dt), D ** -0.5
        return s
    news = _news(case, lens)
    at = [torch.arange(n - t, n, device="cuda") for n, t in zip(lens, news)]
    s["slots"] = torch.cat([s["table"][b][a // page] * page + a % page for b, a in enumerate(at)]).to(torch.int32)
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    if case["fused"]:
        qkv = _normal(gen, (sum(news), 6 * hkv, D), dt)
        s["k"], s["v"] = qkv[:, 4 * hkv:5 * hkv], qkv[:, 5 * hkv:]
    else:
        s["k"], s["v"] = (_rows(gen, (sum(news), hkv, D), dt, channels[i]) for i in range(2))
    return s


def run(s):
    case = s["case"]
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    if not own:
        return {"cache": _plain_cache, "decode": _plain_decode, "linear": _plain_linear}[kind](s)
    import triton_distributed_b200 as tdist
    if kind == "linear":
        x, x_scale = tdist.quantize_int8_rowwise(s["x"])
        return tdist.gemm_int8(x, x_scale, s["w"], s["w_scale"], out_dtype=dt)
    cache = tdist.QuantizedKVCache(s["codes"][0], s["codes"][1], s["scales"][0], s["scales"][1])
    if kind == "cache":
        tdist.kv_cache_write(cache, s["k"], s["v"], s["slots"])
        k, v = tdist.kv_cache_read(cache, s["starts"], s["lens"], s["table"], sum(s["host_lens"]), dt)
        return {"k": k, "v": v}
    return tdist.gqa_fwd_quantized_decode(s["q"], cache, s["lens"], s["table"], window=case["window"] or None, sinks=case["sinks"],
                                          scale=s["scale"], soft_cap=case["soft_cap"])


def _plain_cache(s):
    case, page = s["case"], s["case"]["page"]
    slots = s["slots"].long()
    pages, rows = slots // page, slots % page
    for i, x in enumerate((s["k"], s["v"])):
        codes, scales = _quantise(x, case["bits"])
        s["codes"][i][pages, rows] = codes
        s["scales"][i].transpose(1, 2)[pages, rows] = scales
    dt, out = DTYPES[case["dtype"]], []
    for i in range(2):
        full = torch.empty((sum(s["host_lens"]), case["hkv"], case["head_dim"]), dtype=dt, device="cuda")
        r = 0
        for b, n in enumerate(s["host_lens"]):
            for j in range(0, n, 8192):
                at = torch.arange(j, min(n, j + 8192), device="cuda")
                pages, rows = s["table"][b][at // page].long(), at % page
                full[r + j:r + j + at.numel()] = _values(s["codes"][i][pages, rows], s["scales"][i].transpose(1, 2)[pages, rows], case["bits"])
            r += n
        out.append(full)
    return {"k": out[0], "v": out[1]}


def _keys_of(case, n):
    """Positions that the query of a sequence of n keys sees."""
    lo = max(0, n - case["window"]) if case["window"] else 0
    at = torch.arange(lo, n, device="cuda")
    return torch.cat([torch.arange(0, min(lo, case["sinks"]), device="cuda"), at]) if lo > 0 and case["sinks"] > 0 else at


def _plain_decode(s):
    """Sequence by sequence, some thousand keys at a time: scores of all, one softmax, then the values."""
    case, page, bits = s["case"], s["case"]["page"], s["case"]["bits"]
    hq, hkv, D, cap = case["hq"], case["hkv"], case["head_dim"], case["soft_cap"]
    out = torch.empty_like(s["q"])
    for b, n in enumerate(s["host_lens"]):
        at = _keys_of(case, n)
        pages, rows = s["table"][b][at // page].long(), at % page
        q = s["q"][b].float().view(hkv, hq // hkv, D)
        parts = [slice(j, j + 32768) for j in range(0, at.numel(), 32768)]

        def read(i, part):
            return _values(s["codes"][i][pages[part], rows[part]], s["scales"][i].transpose(1, 2)[pages[part], rows[part]], bits).transpose(0, 1)

        t = torch.cat([torch.matmul(q, read(0, part).transpose(1, 2)) for part in parts], -1) * s["scale"]
        if cap > 0:
            t = cap * torch.tanh(t / cap)
        p = torch.exp(t - t.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        o = sum(torch.matmul(p[..., part], read(1, part)) for part in parts)
        out[b] = o.reshape(hq, D).to(out.dtype)
    return out


def _plain_linear(s):
    """Sums of 1024 products of 8-bit integers are exact in fp32; between them whole numbers."""
    x, w, k = s["x"].float(), s["w"], s["case"]["k"]
    most = x.abs().amax(1, keepdim=True).clamp_min(LEAST)
    codes = torch.round(x * _quotient(127.0, most))
    y = torch.empty((x.shape[0], w.shape[0]), dtype=s["x"].dtype, device="cuda")
    for n0 in range(0, w.shape[0], 16384):
        acc = 0
        for k0 in range(0, k, 1024):
            acc = acc + torch.matmul(codes[:, k0:k0 + 1024], w[n0:n0 + 16384, k0:k0 + 1024].float().t()).to(torch.int32)
        y[:, n0:n0 + 16384] = acc.float() * _quotient(most, 127.0) * s["w_scale"][n0:n0 + 16384]
    return y


def exact(case, seed):
    if work(case)["flops"] > MOST_FLOPS:
        return None
    s = prepare(case, seed)
    if case["kind"] == "linear":
        x = s["x"].double()
        scale = x.abs().amax(1, keepdim=True).clamp_min(LEAST) / 127.0
        x = torch.round(x / scale)
        y = torch.empty((x.shape[0], s["w"].shape[0]), dtype=torch.float64, device="cuda")
        for n0 in range(0, y.shape[1], 4096):
            y[:, n0:n0 + 4096] = (x @ s["w"][n0:n0 + 4096].double().t()) * scale * s["w_scale"][n0:n0 + 4096].double()
        return y
    page, bits, D, hkv = case["page"], case["bits"], case["head_dim"], case["hkv"]

    def stored(i, b, at, h):
        """Rows of head h in 64 bits."""
        pg, rw = s["table"][b].long()[at // page], at % page
        c, p = s["codes"][i][pg, rw, h], s["scales"][i][pg, h, rw].double()
        if bits == 8:
            return (c.double() - 128.0) * p[:, None]
        full = torch.empty((at.numel(), D), dtype=torch.float64, device="cuda")
        full[:, 0::2], full[:, 1::2] = (c % 16).double(), (c // 16).double()
        return full * p[:, :, 0].repeat_interleave(64, 1) + p[:, :, 1].repeat_interleave(64, 1)

    if case["kind"] == "cache":
        out, news = {}, _news(case, s["host_lens"])
        for i, name in enumerate("kv"):
            full = torch.empty((sum(s["host_lens"]), hkv, D), dtype=torch.float64, device="cuda")
            r = t = 0
            for b, n in enumerate(s["host_lens"]):
                old = torch.arange(n - news[b], device="cuda")
                for h in range(hkv):
                    full[r:r + old.numel(), h] = stored(i, b, old, h)
                x = s[name][t:t + news[b]].double()
                if bits == 8:
                    scale = x.abs().amax(-1, keepdim=True).clamp_min(LEAST) / 127.0
                    full[r + old.numel():r + n] = torch.round(x / scale) * scale
                else:
                    for g in range(0, D, 64):
                        y = x[..., g:g + 64]
                        low = _grid(y.amin(-1, keepdim=True), math.floor)
                        size = _grid(((y.amax(-1, keepdim=True) - low) / 15.0).clamp_min(LEAST), math.ceil)
                        full[r + old.numel():r + n, :, g:g + 64] = low + size * torch.round((y - low) / size).clamp(0.0, 15.0)
                r, t = r + n, t + news[b]
            out[name] = full
        return out
    G, cap = case["hq"] // hkv, case["soft_cap"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["host_lens"]):
        at = _keys_of(case, n)
        for h in range(hkv):
            t = s["q"][b, h * G:(h + 1) * G].double() @ stored(0, b, at, h).t() * s["scale"]
            if cap > 0:
                t = cap * torch.tanh(t / cap)
            out[b, h * G:(h + 1) * G] = torch.softmax(t, -1) @ stored(1, b, at, h)
    return out


def _grid(x, way):
    """x (fp64) rounded down or up to the numbers of 8 significant bits."""
    m, e = torch.frexp(x)
    m = m * 256.0
    return torch.ldexp(torch.floor(m) if way is math.floor else torch.ceil(m), e - 8)
