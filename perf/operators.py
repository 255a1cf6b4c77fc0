"""Serving operators over the paged KV cache and the logits, in their plain form and through the library: attention with a
sliding window and sinks (decode and prefill), decode attention of a batch that shares a prefix, and sampling.

`listed()` names the fixed cases, `draw()` gives more of the same ranges, `prepare()` builds what a program holds before the
call, `run()` is one call (`own` false: elementary torch operations in 32 bits; true: the library's operators), `work()` what
it cannot do without, `exact()` the results by the definition in 64 bits.

Kinds of case:
  window_decode   one query token per sequence; it sees the last `window` keys and the first `sinks` (window 0: all)
  window_prefill  a ragged batch of query tokens, the last ones of their sequences; position p sees the keys j <= p with
                  j > p - window or j < sinks (window 0: all j <= p)
  prefix_decode   one query token per sequence over the keys of one prefix that all share, and the sequence's own
  sample          one token per row of logits: temperature, top-k, top-p, min-p, then the inverse of the cumulative weights
                  in the order of the tokens at a given uniform number. Weights are whole multiples of 2^-31 of the largest
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HEADS = ((16, 16), (32, 8), (64, 8), (6, 1), (96, 12))
MOST_FLOPS = 2.2e12   # about the largest listed case
MOST_BYTES = 4.5e9    # of inputs
ONE = 2147483648.0    # weight of a row's largest logit


def _window_decode(B, hq, hkv, head_dim, kv, page, window, sinks, dtype="bf16", ragged=False, soft_cap=0.0):
    return dict(kind="window_decode", B=B, hq=hq, hkv=hkv, head_dim=head_dim, kv=kv, page=page, window=window, sinks=sinks,
                dtype=dtype, ragged=ragged, soft_cap=soft_cap)


def _window_prefill(B, hq, hkv, head_dim, new, kv, page, window, sinks, dtype="bf16", ragged=False, soft_cap=0.0, fused=False):
    return dict(kind="window_prefill", B=B, hq=hq, hkv=hkv, head_dim=head_dim, new=new, kv=kv, page=page, window=window,
                sinks=sinks, dtype=dtype, ragged=ragged, soft_cap=soft_cap, fused=fused)


def _prefix_decode(B, hq, hkv, head_dim, prefix, kv, page, dtype="bf16", ragged=True, soft_cap=0.0):
    return dict(kind="prefix_decode", B=B, hq=hq, hkv=hkv, head_dim=head_dim, prefix=prefix, kv=kv, page=page, dtype=dtype,
                ragged=ragged, soft_cap=soft_cap)


def _sample(B, vocab, dtype="bf16", filters="mixed"):
    return dict(kind="sample", B=B, vocab=vocab, dtype=dtype, filters=filters)


def listed():
    return [
        # one interactive request in a windowed layer: launch latency decides
        dict(name="window_decode_b1", **_window_decode(1, 32, 8, 128, 4096, 16, 1024, 4)),
        # a serving batch of long conversations of all lengths, the window bounds what each reads
        dict(name="window_decode_b64_ragged", **_window_decode(64, 64, 8, 128, 16384, 64, 4096, 4, dtype="fp16", ragged=True)),
        # a few short chunks of ragged requests, q a part of a fused projection
        dict(name="window_prefill_small", **_window_prefill(5, 64, 8, 64, 77, 1000, 16, 128, 4, ragged=True, fused=True)),
        # a 2048-token chunk of one long prompt
        dict(name="window_prefill_chunk", **_window_prefill(1, 32, 8, 128, 2048, 8192, 16, 4096, 4)),
        # a long prompt at once
        dict(name="window_prefill_16k", **_window_prefill(1, 64, 8, 128, 16384, 16384, 64, 4096, 4)),
        # a batch of ragged prompts through a full layer (no window), soft cap, heads of 64
        dict(name="full_prefill_ragged", **_window_prefill(7, 32, 8, 64, 3001, 3001, 16, 0, 0, dtype="fp16", ragged=True, soft_cap=30.0)),
        # a few requests on one short system prompt
        dict(name="prefix_b8_2k", **_prefix_decode(8, 32, 8, 128, 2048, 256, 16)),
        # a serving batch on one long document
        dict(name="prefix_b64_32k", **_prefix_decode(64, 32, 8, 128, 32768, 1024, 16)),
        # many samples of one prompt, odd sizes, large heads of one kv head
        dict(name="prefix_b201_odd", **_prefix_decode(201, 6, 1, 256, 5003, 300, 16, dtype="fp16")),
        # one interactive request's token
        dict(name="sample_b1_32k", **_sample(1, 32000, "fp32")),
        # a serving batch's tokens, each request with its own settings
        dict(name="sample_b64_128k", **_sample(64, 128256, "bf16")),
        # a large batch over an odd vocabulary
        dict(name="sample_b256_odd", **_sample(256, 100003, "fp32")),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread evenly over the logarithm."""
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("window_decode", "window_prefill", "window_prefill", "prefix_decode", "prefix_decode", "sample", "sample"))
    while True:
        hq, hkv = rng.choice(HEADS)
        head_dim, page = rng.choice((64, 128, 128, 256)), rng.choice((1, 16, 16, 64))
        dtype, cap = rng.choice(("bf16", "fp16")), rng.choice((0.0, 0.0, 30.0))
        window, sinks = _log(rng, 16, 8192), rng.choice((0, 1, 4, 4, 37))
        if rng.random() < 0.15:
            window = 0
        if kind == "window_decode":
            case = _window_decode(_log(rng, 1, 64), hq, hkv, head_dim, _log(rng, 1, 65536), page, window, sinks, dtype,
                                  rng.random() < 0.5, cap)
        elif kind == "window_prefill":
            new = _log(rng, 1, 8192)
            case = _window_prefill(_log(rng, 1, 16), hq, hkv, head_dim, new, _log(rng, new, 65536), page, window, sinks, dtype,
                                   rng.random() < 0.5, cap, rng.random() < 0.5)
        elif kind == "prefix_decode":
            case = _prefix_decode(_log(rng, 1, 256), hq, hkv, head_dim, _log(rng, 16, 131072), _log(rng, 1, 2048), page, dtype,
                                  rng.random() < 0.8, cap)
        else:
            case = _sample(_log(rng, 1, 256), _log(rng, 1000, 200000), rng.choice(("bf16", "fp16", "fp32")),
                           rng.choice(("mixed", "mixed", "none", "top_k", "top_p", "min_p", "greedy")))
        if work(case)["flops"] <= MOST_FLOPS and _held(case) <= MOST_BYTES:
            return case


def _lens(case):
    """Per sequence: query tokens and keys, on the host. Ragged: evenly spread up to the largest."""
    B, kv, kind = case["B"], case["kv"], case["kind"]
    if kind == "window_prefill":
        new = [max(1, case["new"] * (i + 1) // B) if case["ragged"] else case["new"] for i in range(B)]
        # the chunk that ends its sequence; of ragged ones each has its own context before it
        before = kv - case["new"]
        return [(n, n + (before * ((i * 5 + 2) % B + 1) // B if case["ragged"] else before)) for i, n in enumerate(new)]
    return [(1, max(1, kv * (i + 1) // B) if case["ragged"] else kv) for i in range(B)]


def _pages(case):
    """Pages of the longest sequence, and of the prefix."""
    return -(-max(n for _, n in _lens(case)) // case["page"]), -(-case.get("prefix", 0) // case["page"])


def _held(case):
    """Bytes of the caches (or logits) that a state holds."""
    if case["kind"] == "sample":
        return 1.0 * case["B"] * case["vocab"] * (4 if case["dtype"] == "fp32" else 2)
    per_seq, prefix = _pages(case)
    return 4.0 * (case["B"] * per_seq + prefix) * case["page"] * case["hkv"] * case["head_dim"]


def _visible(pos, case):
    """Keys that a query at position `pos` sees."""
    w, s = case["window"], case["sinks"]
    return pos + 1 if w == 0 else min(pos + 1, w + min(s, max(0, pos + 1 - w)))


def _pairs(n, kv, case):
    """Visible (query, key) pairs of the last n positions of kv."""
    w, s = case["window"], case["sinks"]
    if w == 0 or n <= 64:
        return sum(_visible(p, case) for p in range(kv - n, kv)) if n <= 64 else n * (kv - n) + n * (n + 1) // 2
    return sum(_visible(p, case) for p in range(kv - n, min(kv, max(kv - n, w + s)))) + max(0, kv - max(kv - n, w + s)) * (w + s)


def _normal(gen, shape, dtype, scale=1.0):
    t = torch.empty(shape, dtype=torch.float32, device="cuda").normal_(generator=gen) if dtype == torch.float32 else \
        torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)
    return t if scale == 1.0 else t.mul_(scale)


def _settings(case, seed):
    """Per row: temperature, top-k, top-p and min-p as requests set them; most set one or two of them."""
    rng = random.Random(int(seed) * 7 + 1)
    rows = []
    for _ in range(case["B"]):
        which = case["filters"]
        if which == "mixed":
            which = rng.choice(("none", "top_k", "top_p", "top_p", "min_p", "greedy", "all"))
        t = 0.0 if which == "greedy" else rng.choice((0.6, 0.8, 1.0, 1.0, 1.3))
        k = rng.choice((1, 20, 50, 1000)) if which in ("top_k", "all") else 0
        p = rng.choice((0.5, 0.9, 0.95, 0.99)) if which in ("top_p", "all") else 1.0
        m = rng.choice((0.01, 0.05, 0.1)) if which in ("min_p", "all") else 0.0
        rows.append((t, k, p, m))
    return rows


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s, B, dt = {"case": dict(case)}, case["B"], DTYPES[case["dtype"]]
    if case["kind"] == "sample":
        V = case["vocab"]
        s["logits"] = _normal(gen, (B, V), dt, 2.5)
        # every fourth row only admits the tokens that a grammar allows: the others are -inf
        if B > 1:
            s["logits"][::4, ::3] = float("-inf")
        s["u"] = torch.rand(B, generator=gen, device="cuda")
        rows = _settings(case, seed)
        s["temperature"] = torch.tensor([r[0] for r in rows], device="cuda")
        s["top_k"] = torch.tensor([r[1] for r in rows], dtype=torch.int32, device="cuda")
        s["top_p"] = torch.tensor([r[2] for r in rows], device="cuda")
        s["min_p"] = torch.tensor([r[3] for r in rows], device="cuda")
        return s
    hq, hkv, D, page = case["hq"], case["hkv"], case["head_dim"], case["page"]
    per_seq, prefix = _pages(case)
    pages = B * per_seq + prefix
    s["k"], s["v"] = _normal(gen, (pages, page, hkv, D), dt), _normal(gen, (pages, page, hkv, D), dt)
    # pages as a running server hands them out: in no order
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    s["table"], s["prefix_table"] = order[:B * per_seq].view(B, per_seq), order[B * per_seq:]
    lens = _lens(case)
    random.Random(int(seed)).shuffle(lens)   # lengths in no order either
    s["host_lens"] = lens
    s["lens"] = torch.tensor([n for _, n in lens], dtype=torch.int32, device="cuda")
    total = sum(n for n, _ in lens)
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    s["host_starts"], s["starts"] = starts, torch.tensor(starts, dtype=torch.int32, device="cuda")
    if case.get("fused"):
        s["q"] = _normal(gen, (total, hq + 2 * hkv, D), dt)[:, :hq]
    else:
        s["q"] = _normal(gen, (total, hq, D), dt)
    s["scale"] = D ** -0.5
    if "prefix" in case:
        s["prefix_len"] = torch.tensor([case["prefix"]], dtype=torch.int32, device="cuda")
    return s


def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        return {"window_decode": _plain_window, "window_prefill": _plain_window, "prefix_decode": _plain_prefix,
                "sample": _plain_sample}[kind](s)
    import triton_distributed_b200 as tdist
    if kind == "sample":
        tokens, logprobs, log_norm = tdist.sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                                         top_p=s["top_p"], min_p=s["min_p"])
        return {"tokens": tokens, "logprobs": logprobs, "log_norm": log_norm}
    if kind == "window_decode":
        return tdist.gqa_fwd_window_decode(s["q"], s["k"], s["v"], s["lens"], s["table"], window=case["window"] or None,
                                           sinks=case["sinks"], scale=s["scale"], soft_cap=case["soft_cap"])
    if kind == "window_prefill":
        return tdist.gqa_fwd_window_prefill(s["q"], s["k"], s["v"], s["starts"], s["lens"], s["table"], window=case["window"] or None,
                                            sinks=case["sinks"], scale=s["scale"], soft_cap=case["soft_cap"])
    return tdist.gqa_fwd_shared_prefix_decode(s["q"], s["k"], s["v"], s["prefix_len"], s["prefix_table"], s["lens"], s["table"],
                                              scale=s["scale"], soft_cap=case["soft_cap"])


def _capped(scores, case):
    return case["soft_cap"] * torch.tanh(scores / case["soft_cap"]) if case["soft_cap"] > 0 else scores


def _plain_window(s):
    """Sequence by sequence and some hundred queries at a time: the keys from the first one's window on, and the sinks before."""
    case, page = s["case"], s["case"]["page"]
    hkv, D, G, w = case["hkv"], case["head_dim"], case["hq"] // case["hkv"], case["window"]
    out = torch.empty(s["q"].shape, dtype=s["q"].dtype, device="cuda")
    step = max(1, min(512, (1 << 28) // (case["hq"] * (w + 512 if w else case["kv"]))))
    for b, (n, kv) in enumerate(s["host_lens"]):
        for i0 in range(0, n, step):
            i1 = min(n, i0 + step)
            first, last = kv - n + i0, kv - n + i1 - 1           # positions of the queries
            lo = max(0, first - w + 1) if w else 0
            at = torch.arange(lo, last + 1, device="cuda")
            if lo > 0 and case["sinks"] > 0:
                at = torch.cat([torch.arange(0, min(lo, case["sinks"]), device="cuda"), at])
            pages, rows = s["table"][b][at // page].long(), at % page
            k, v = s["k"][pages, rows].float(), s["v"][pages, rows].float()   # [keys, hkv, D]
            pos = torch.arange(first, last + 1, device="cuda").view(-1, 1)
            seen = at.view(1, -1) <= pos
            if w:
                seen = seen & ((at.view(1, -1) > pos - w) | (at.view(1, -1) < case["sinks"]))
            q = s["q"][s["host_starts"][b] + i0:s["host_starts"][b] + i1].float().view(i1 - i0, hkv, G, D)
            t = torch.matmul(q.permute(1, 2, 0, 3).reshape(hkv, G * (i1 - i0), D), k.permute(1, 2, 0)) * s["scale"]
            t = _capped(t, case).view(hkv, G, i1 - i0, -1).masked_fill(~seen, float("-inf"))
            p = torch.exp(t - t.amax(-1, keepdim=True))
            p = (p / p.sum(-1, keepdim=True)).view(hkv, G * (i1 - i0), -1)
            o = torch.matmul(p, v.permute(1, 0, 2)).view(hkv, G, i1 - i0, D)
            out[s["host_starts"][b] + i0:s["host_starts"][b] + i1] = o.permute(2, 0, 1, 3).reshape(i1 - i0, case["hq"], D).to(out.dtype)
    return out


def _plain_prefix(s):
    """The prefix' scores for all sequences in one product, the own keys padded to the longest; one softmax over both."""
    case, page = s["case"], s["case"]["page"]
    B, hq, hkv, D, P = case["B"], case["hq"], case["hkv"], case["head_dim"], case["prefix"]
    G, most = hq // hkv, max(n for _, n in s["host_lens"])
    at = torch.arange(P, device="cuda")
    pages, rows = s["prefix_table"][at // page].long(), at % page
    kp, vp = s["k"][pages, rows].float(), s["v"][pages, rows].float()                # [P, hkv, D]
    at = torch.arange(most, device="cuda")
    mine = at.view(1, -1) < s["lens"].view(-1, 1)
    pages, rows = s["table"][:, at // page].long(), at % page
    out = torch.empty((B, hq, D), dtype=s["q"].dtype, device="cuda")
    q = s["q"].float().view(B, hkv, G, D)
    for h in range(hkv):
        ks, vs = s["k"][pages, rows, h].float(), s["v"][pages, rows, h].float()      # [B, most, D]
        vs = vs.masked_fill(~mine.unsqueeze(-1), 0.0)
        tp = _capped(torch.matmul(q[:, h].reshape(B * G, D), kp[:, h].t()) * s["scale"], case).view(B, G, P)
        ts = _capped(torch.matmul(q[:, h], ks.transpose(1, 2)) * s["scale"], case).masked_fill(~mine.unsqueeze(1), float("-inf"))
        top = torch.maximum(tp.amax(-1, keepdim=True), ts.amax(-1, keepdim=True))
        tp, ts = torch.exp(tp - top), torch.exp(ts - top)
        o = torch.matmul(tp.view(B * G, P), vp[:, h]).view(B, G, D) + torch.matmul(ts, vs)
        out[:, h * G:(h + 1) * G] = (o / (tp.sum(-1, keepdim=True) + ts.sum(-1, keepdim=True))).to(out.dtype)
    return out


def _plain_sample(s):
    x = s["logits"].float()
    V = x.shape[1]
    x = torch.where(torch.isnan(x), float("-inf"), x) + 0.0
    temperature, top_k = s["temperature"], s["top_k"].long()
    greedy = temperature <= 0
    inv = 1.0 / torch.where(greedy, 1.0, temperature)
    top = x.amax(1)
    y = torch.where(x == top.view(-1, 1), 0.0, (x - top.view(-1, 1)) * inv.view(-1, 1))
    w = torch.round(torch.exp(y) * ONE).long()
    # by weight, ties by number: every filter keeps the first ones of this order
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    sorted_w = w.gather(1, order)
    rank = torch.arange(V, device="cuda").view(1, -1)
    k = torch.where(greedy, 1, torch.where(top_k <= 0, V, top_k)).view(-1, 1)
    keep = rank < k
    before = torch.cumsum(sorted_w, 1) - sorted_w
    mass = (sorted_w * keep).sum(1)
    limit = torch.ceil(s["top_p"].double() * mass.double()).clamp_min(1.0).long().view(-1, 1)
    keep = keep & ((before < limit) | (s["top_p"] >= 1).view(-1, 1))
    least = torch.ceil(s["min_p"].double().clamp(0.0, 1.0) * ONE).long().view(-1, 1)
    keep = keep & (sorted_w >= least)
    kept = torch.zeros_like(w).scatter_(1, order, sorted_w * keep)
    mass = kept.sum(1)
    target = torch.minimum(torch.floor(s["u"].double() * mass.double()).long(), mass - 1).view(-1, 1)
    tokens = (torch.cumsum(kept, 1) > target).to(torch.int8).argmax(1)
    norm = torch.log(mass.float() / ONE)
    none = top == float("-inf")
    logprobs = y.gather(1, tokens.view(-1, 1)).view(-1) - norm
    return {"tokens": torch.where(none, -1, tokens).to(torch.int32), "logprobs": torch.where(none, float("-inf"), logprobs),
            "log_norm": torch.where(none, float("-inf"), top * inv + norm)}


def work(case):
    if case["kind"] == "sample":
        n = 1.0 * case["B"] * case["vocab"]
        return {"bytes": n * (4 if case["dtype"] == "fp32" else 2) + 32.0 * case["B"], "flops": 4.0 * n}
    hq, hkv, D, lens = case["hq"], case["hkv"], case["head_dim"], _lens(case)
    rows = sum(n for n, _ in lens)
    if case["kind"] == "prefix_decode":
        keys = sum(n for _, n in lens)
        seen, pairs = keys + case["prefix"], keys + case["B"] * case["prefix"]
    else:
        pairs = sum(_pairs(n, kv, case) for n, kv in lens)
        # keys that some query sees: from the first query's window on, and the sinks before
        seen = sum(_visible(kv - n, case) + n - 1 for n, kv in lens)
    return {"bytes": 4.0 * seen * hkv * D + 4.0 * rows * hq * D, "flops": 4.0 * pairs * hq * D}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        return _exact_sample(s)
    if work(case)["flops"] > MOST_FLOPS:
        return None
    page, hkv, D, w, cap = case["page"], case["hkv"], case["head_dim"], case.get("window", 0), case["soft_cap"]
    G = case["hq"] // hkv
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, (n, kv) in enumerate(s["host_lens"]):
        pages = [s["table"][b, :-(-kv // page)].long()]
        k = [s["k"][pages[0]].flatten(0, 1)[:kv]]
        v = [s["v"][pages[0]].flatten(0, 1)[:kv]]
        shared = case.get("prefix", 0)
        if shared:
            pre = s["prefix_table"].long()
            k.insert(0, s["k"][pre].flatten(0, 1)[:shared])
            v.insert(0, s["v"][pre].flatten(0, 1)[:shared])
        k, v = torch.cat(k), torch.cat(v)
        keys = torch.arange(shared + kv, device="cuda")
        for h in range(hkv):
            kh, vh = k[:, h].double(), v[:, h].double()
            for i0 in range(0, n, 256):
                i1 = min(n, i0 + 256)
                pos = shared + kv - n + torch.arange(i0, i1, device="cuda").unsqueeze(1)
                c0 = int(max(0, shared + kv - n + i0 - w + 1)) if w else 0   # keys before it are sinks or nobody's
                c1 = shared + kv - n + i1
                part = keys[c0:c1] if case.get("sinks", 0) == 0 or c0 == 0 else torch.cat([keys[:min(c0, case["sinks"])], keys[c0:c1]])
                hidden = part > pos
                if w:
                    hidden = hidden | ((part <= pos - w) & (part >= case["sinks"]))
                rows = slice(s["host_starts"][b] + i0, s["host_starts"][b] + i1)
                for g in range(h * G, (h + 1) * G):
                    t = s["q"][rows, g].double() @ kh[part].t() * s["scale"]
                    if cap > 0:
                        t = cap * torch.tanh(t / cap)
                    t[hidden] = float("-inf")
                    out[rows, g] = torch.softmax(t, -1) @ vh[part]
    return out


def _exact_sample(s):
    """The log of the kept tokens' mass, row by row. Which token a number falls on, and so its probability, goes by the
    whole-number weights: no 64-bit value."""
    x, rows = s["logits"].double(), []
    for b in range(x.shape[0]):
        t, k, p, m = (float(s[n][b]) for n in ("temperature", "top_k", "top_p", "min_p"))
        z = torch.sort(x[b] / t if t > 0 else x[b], descending=True).values
        z = z[:1] if t <= 0 else (z[:int(k)] if k > 0 else z)
        prob = torch.softmax(z, 0)
        if p < 1:
            z = z[:int((torch.cumsum(prob, 0) < p).sum()) + 1]
        z = z[z >= z[0] + (math.log(m) if m > 0 else -math.inf)]
        rows.append(torch.logsumexp(z, 0))
    return {"tokens": None, "logprobs": None, "log_norm": torch.stack(rows)}
