"""Attention over a quantised cache where weights, values and scores lie far apart, against 64 bits.

Bound per element, with p the weights relative to the largest, l their sum, A = sum p |v| / l:
* half a step of the result's type, of itself (fp16: or half of its least step, 2^-25; results beyond its largest are infinite)
* a weight times its value's scale (a group's step) is rounded to fp16: 2^-11 of itself, or 2^-25 of a unit that is at most 2^-5 of the largest such product of
  that group; codes reach 127 (8): per key 2^-30 max_j(p_j scale_j) 127 / l (4 bits: 8 step for 127 scale)
* scores move weights and their sum: the query's share max|q| / 32640 sum |k_d| scale, 2^-23 (D / 16 + 6) of sum |q_d k_d| scale, the exponential 2^-20; sums of n / 16 fp32 steps
"""
import math

import pytest
import torch

import triton_distributed_b200 as tdist
from test_quantized_edges_cpu import largest_rows, wide_rows

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _cache(k, v, bits, page=16):
    """A sequence [n, Hkv, D] in a cache of its own, on the CPU, and its table."""
    n, Hkv, D = k.shape
    pages = -(-n // page)
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(n)).to(torch.int32).view(1, -1)
    cache = tdist.create_quantized_kv_cache(pages, page, Hkv, D, bits, "cpu")
    at = torch.arange(n)
    tdist.kv_cache_write(cache, k, v, table[0].long()[at // page] * page + at % page)
    return cache, table


def _rows(cache, table, at, i):
    """What is stored at the positions of a sequence, in 64 bits: [Hkv, n, D]; |step c| + |least| of each; the product's size per unit of weight [Hkv, n, D]."""
    page = cache.k.shape[1]
    pages, rows = table[at // page].long(), at % page
    c, s = cache[i][pages, rows].transpose(0, 1), cache[2 + i].transpose(1, 2)[pages, rows].double().transpose(0, 1)
    if cache.bits == 8:
        v = (c.double() - 128.0) * s.unsqueeze(-1)
        return v, v.abs(), (127.0 * s).unsqueeze(-1).expand_as(v)
    c = torch.stack([c & 15, c >> 4], -1).flatten(-2).double().unflatten(-1, (-1, 64))
    step, least = s[..., 0:1], s[..., 1:2]
    return (c * step + least).flatten(-2), (c * step + least.abs()).flatten(-2), (8.0 * step).expand_as(c).flatten(-2)


def _check(q, cache, table, n, scale=None, query=1 / 32640, **kw):
    """A sequence of n keys."""
    gpu = q.cuda(), tdist.QuantizedKVCache(*(t.cuda() for t in cache)), torch.tensor([n], dtype=torch.int32).cuda(), table.cuda()
    _compare(tdist.gqa_fwd_quantized_decode(*gpu, scale=scale, **kw).cpu(), q, cache, table, [n], scale, query)


def _compare(got, q, cache, table, lens, scale=None, query=1 / 32640, window=None, sinks=0):
    D, Hkv = q.shape[2], cache.k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    for b, n in enumerate(lens):
        lo = 0 if window is None else max(0, n - window)
        at = torch.cat([torch.arange(0, min(sinks, lo)), torch.arange(lo, n)])
        if at.numel() == 0:
            assert (got[b] == 0).all()
            continue
        (k, ka, _), (v, va, size) = _rows(cache, table[b], at, 0), _rows(cache, table[b], at, 1)
        qq = q[b].double().view(Hkv, -1, D)
        t = qq @ k.transpose(1, 2) * scale
        p = torch.exp(t - t.amax(-1, keepdim=True))
        l = p.sum(-1, keepdim=True)
        ref, A = p @ v / l, p @ va / l
        # a score's error counts with the key's weight: what weighs nothing may be off by much
        off = query * qq.abs().amax(-1, keepdim=True) * ka.sum(-1).unsqueeze(1) * abs(scale) + (D / 16 + 6) * 2.0 ** -23 * (qq.abs() @ ka.transpose(1, 2)) * abs(scale)
        moved = (p * torch.expm1(off + 2.0 ** -20)) @ va / l + (p * torch.expm1(off + 2.0 ** -20)).sum(-1, keepdim=True) / l * A
        least = torch.stack([(p * size[..., d].unsqueeze(1)).amax(2, keepdim=True).expand(-1, -1, 64) for d in range(0, D, 64)], 2).flatten(2) * at.numel() * 2.0 ** -30 / l
        tol = HALF[q.dtype] * ref.abs() + 1.01 * ((2.0 ** -11 + at.numel() / 16 * 2.0 ** -23) * A + moved + least) + (2.0 ** -25 if q.dtype == torch.float16 else 2.0 ** -120)
        out, most = got[b].double().view(Hkv, -1, D), torch.finfo(q.dtype).max
        inf = out.abs() == math.inf               # where the bound reaches beyond the type's range, and has to where it lies beyond
        assert bool((out == ref.sign() * math.inf)[inf].all()) and bool((ref.abs() + tol > most)[inf].all()) and bool(inf[ref.abs() - tol > most].all())
        err = (out - ref).abs().masked_fill(inf, 0.0)
        assert bool((err <= tol).all()), (b, n, float(err.max()), float((err / tol).max()))


def _keys(n, G, D, scores, seed):
    """Query heads of one kind and keys whose scores (scale 1 / D) are about `scores`, with some noise."""
    g = torch.Generator().manual_seed(seed)
    q = torch.where(torch.rand(1, 1, D, generator=g) < 0.5, -1.0, 1.0).expand(1, G, D) * (1.0 + torch.arange(G).view(1, G, 1) / 64)
    k = q[:, :1] * scores.view(n, 1, 1) + 0.3 * torch.randn(n, 1, D, generator=g)
    return q, k, torch.randn(n, 1, D, generator=g)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("split", [0, 1, 3, 40])
@pytest.mark.parametrize("D,G,n", [(64, 3, 200), (128, 4, 700), (128, 12, 333), (256, 6, 500)])
@pytest.mark.parametrize("where", ["first", "middle", "last"])
def test_a_large_value_without_weight(bits, dtype, split, D, G, n, where):
    """One value 2^30 times the others, at a key that weighs e^-60: the others' sum is the result."""
    at = {"first": 0, "middle": n // 2, "last": n - 1}[where]
    scores = torch.zeros(n)
    scores[at] = -60.0
    q, k, v = _keys(n, G, D, scores, n + D)
    v[at] *= 2.0 ** 30
    _check(q.to(dtype).contiguous(), *_cache(k.bfloat16(), v.bfloat16(), bits), n, scale=1.0 / D, kv_split=split)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("split", [0, 1])
@pytest.mark.parametrize("gap,ratio", [(60.0, 30), (20.8, 30), (5.0, 30), (60.0, 80), (0.5, 20)])
@pytest.mark.parametrize("least", [-60.0, 0.0])
def test_scores_rise_past_large_values(bits, dtype, split, gap, ratio, least):
    """Tile by tile scores rise by `gap` and values shrink by 2^ratio, down to 2^least: what was the largest product comes to nothing, or does not."""
    n, D = 512, 128
    step = torch.arange(n) // 96                # every warp of 6 takes part in each
    q, k, v = _keys(n, 4, D, gap * step.float(), 3)
    v = v * torch.exp2(60.0 - ratio * step.float()).clamp_min(2.0 ** least).view(n, 1, 1)
    _check(q.to(dtype).contiguous(), *_cache(k.bfloat16(), v.bfloat16(), bits), n, scale=1.0 / D, kv_split=split)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,G", [(128, 4), (128, 16), (256, 8)])
def test_groups_of_values_far_apart(dtype, D, G):
    """4 bits: the dimensions of one group are 2^40 times those of another, which keeps its own."""
    n = 300
    q, k, v = _keys(n, G, D, torch.zeros(n), 5)
    v = v * torch.exp2(40.0 * (torch.arange(D) // 64 % 2))
    v[7, 0, :64] *= 2.0 ** 60
    for j in (0, 64):
        w = v.clone()
        w[:, :, j:j + 64] *= 2.0 ** -40
        _check(q.to(dtype).contiguous(), *_cache(k.bfloat16(), w.bfloat16(), 4), n, scale=1.0 / D)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_long_tail_of_small_weights(bits, dtype):
    """One key of most of the weight whose value is nearly zero, and 65536 keys of 2^-26 each whose values are alike: their sum is the result."""
    n, D = 65537, 64
    scores = torch.full((n,), -26 * math.log(2.0))
    scores[100] = 0.0
    q, k, v = _keys(n, 2, D, scores, 6)
    k = q[:, :1] * scores.view(n, 1, 1) + 0.0 * k
    v = 1.0 + 0.01 * v
    v[100] = 2.0 ** -20
    _check(q.to(dtype).contiguous(), *_cache(k.bfloat16(), v.bfloat16(), bits), n, scale=1.0 / D, kv_split=8)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_queries_whose_elements_are_exact(bits, dtype):
    """No element more than 2^6 (bf16, 8 significant bits) or 2^3 (fp16, 11) below the largest, whatever its leading bits: nothing is rounded."""
    n, D, G = 300, 128, 4
    g = torch.Generator().manual_seed(20)
    most = 64.0 if dtype == torch.bfloat16 else 8.0
    for lead in (1.0, 1.5, 255 / 128):
        q = ((1 + torch.rand(1, G, D, generator=g)) * torch.where(torch.rand(1, G, D, generator=g) < 0.5, -1.0, 1.0)).clamp(-1.9, 1.9)
        q[:, :, 5] = most * lead
        k, v = (torch.randn(n, 1, D, generator=g) for _ in range(2))
        k = 8 * k
        k[:, :, 5] *= 0.01
        _check(q.to(dtype), *_cache(k.bfloat16(), v.bfloat16(), bits), n, query=0.0)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("size,scale", [(2.0 ** 124, 2.0 ** -126), (2.0 ** 125, 2.0 ** -126), (2.0 ** -95, 2.0 ** 90)])
def test_queries_near_the_ends_of_bf16(bits, size, scale):
    """Elements above 2^126, and tiny ones, with a scale that makes scores of ordinary size."""
    n, D = 200, 64
    g = torch.Generator().manual_seed(21)
    q = torch.randn(1, 4, D, generator=g)
    q = (q / q.abs().amax() * 3.98 * size).to(torch.bfloat16)
    k, v = (torch.randn(n, 1, D, generator=g) for _ in range(2))
    _check(q, *_cache(k.bfloat16(), v.bfloat16(), bits), n, scale=scale)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size,keys,scale", [(1.0, 2.0 ** 122, 2.0 ** -125), (2.0 ** -8, 2.0 ** 122, 2.0 ** -117), (2.0 ** 8, 2.0 ** 110, 2.0 ** -121), (2.0 ** 8, 2.0 ** -80, 2.0 ** 69),
                                             (2.0 ** -80, 2.0 ** 77, None), (2.0 ** 77, 2.0 ** -80, None), (2.0 ** 121, 2.0 ** -90, 2.0 ** -34), (2.0 ** -90, 2.0 ** 122, 2.0 ** -35),
                                             (2.0 ** -70, 2.0 ** -70, 2.0 ** 127), (2.0 ** 60, 2.0 ** 62, 2.0 ** -125)])
def test_scores_of_ordinary_size_from_far_apart(bits, dtype, size, keys, scale):
    """What is large and what is small come together only in the score."""
    if dtype == torch.float16 and not 2.0 ** -9 < size < 2.0 ** 9:
        size, scale = 2.0 ** -8, (64 ** -0.5 if scale is None else scale) * size * 2.0 ** 8
        if not 2.0 ** -126 <= scale < 2.0 ** 127:
            pytest.skip("fp16 queries of that size need a scale that fp32 does not have")
    n, D = 200, 64
    g = torch.Generator().manual_seed(22)
    q = torch.randn(1, 4, D, generator=g) * size
    k, v = (torch.randn(n, 1, D, generator=g) for _ in range(2))
    _check(q.to(dtype), *_cache((k * keys).bfloat16(), v.bfloat16(), bits), n, scale=scale)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("cap", [1e-10, 2.0 ** -61, 1e-38, 1e-39, 1e-44, 1e30, 2.0 ** 127])
def test_caps_of_any_size(bits, cap):
    """A tiny cap (subnormal ones too): the mean of the values. A huge one: as none, up to the cap's own arithmetic."""
    n, D = 300, 64
    g = torch.Generator().manual_seed(23)
    q, (k, v) = torch.randn(1, 4, D, generator=g).to(torch.bfloat16), (torch.randn(n, 1, D, generator=g).to(torch.bfloat16) for _ in range(2))
    cache, table = _cache(k, v, bits)
    gpu = q.cuda(), tdist.QuantizedKVCache(*(t.cuda() for t in cache)), torch.tensor([n], dtype=torch.int32).cuda(), table.cuda()
    got = tdist.gqa_fwd_quantized_decode(*gpu, soft_cap=cap).cpu()
    if cap > 1.0:
        _compare(got, q, cache, table, [n])
    else:
        _compare(got, torch.zeros_like(q), cache, table, [n])


# ---------------------------------------------------------------------------- writing
@pytest.mark.parametrize("heads", [1, 3])
def test_groups_whose_range_is_beyond_fp32_are_the_statement_bit_for_bit(heads):
    x = torch.cat([wide_rows(), wide_rows().flip(0), torch.randn(8, 1, 64).to(torch.bfloat16)], 1)[:, :heads].contiguous()
    cpu = tdist.create_quantized_kv_cache(1, 8, heads, 64, 4, "cpu")
    gpu = tdist.QuantizedKVCache(*(t.cuda() for t in cpu))
    tdist.kv_cache_write(cpu, x, x, torch.arange(8))
    tdist.kv_cache_write(gpu, x.cuda(), x.cuda(), torch.arange(8).cuda())
    for a, b in zip(cpu, gpu):
        assert torch.equal(a.view(torch.uint8), b.cpu().view(torch.uint8))


# ---------------------------------------------------------------------------- reading
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("into", [torch.bfloat16, torch.float16])
def test_largest_numbers_are_read_as_the_statement_has_them(bits, dtype, into):
    x = torch.cat([largest_rows(dtype), wide_rows().to(dtype).clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max)])
    x[-1, 0, 3], x[-2, 0, 4] = math.nan, math.inf
    n = x.shape[0]
    cpu = tdist.create_quantized_kv_cache(1, n, 1, 64, bits, "cpu")
    tdist.kv_cache_write(cpu, x, x.flip(0), torch.arange(n))
    gpu = tdist.QuantizedKVCache(*(t.cuda() for t in cpu))
    args = torch.tensor([0, n]), torch.tensor([n]), torch.tensor([[0]])
    for a, b in zip(tdist.kv_cache_read(cpu, *args, n, into), tdist.kv_cache_read(gpu, *(t.cuda() for t in args), n, into)):
        b = b.cpu()
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0.0, math.inf, -math.inf), b.nan_to_num(0.0, math.inf, -math.inf))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("first", [-5, -(1 << 31), -(1 << 40)])
def test_sequences_that_start_before_row_0_are_not_read(bits, first):
    """As in the statement; with pages of one token and the lowest start a row's distance from it would pass 31 bits."""
    x = torch.randn(40, 2, 64, generator=torch.Generator().manual_seed(30)).to(torch.bfloat16)
    cpu = tdist.create_quantized_kv_cache(40, 1, 2, 64, bits, "cpu")
    tdist.kv_cache_write(cpu, x, x, torch.arange(40))
    gpu = tdist.QuantizedKVCache(*(t.cuda() for t in cpu))
    for starts in ([first, 7, 20], [first, first + 3, 12], [first, first, first]):
        args = torch.tensor(starts), torch.tensor([(1 << 31) - 1, 9]), torch.arange(40).view(2, 20)
        want, got = tdist.kv_cache_read(cpu, *args, 24), tdist.kv_cache_read(gpu, *(t.cuda() for t in args), 24)
        for a, b in zip(want, got):
            assert torch.equal(a, b.cpu())


# ---------------------------------------------------------------------------- as it is chosen
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,Hq,Hkv,D,page,most,window,sinks", [
    (70, 8, 2, 128, 16, 9000, None, 0),       # equal shares of many ragged sequences
    (1, 16, 8, 64, 16, 150000, None, 0),      # of a long one
    (3, 10, 1, 256, 7, 40000, None, 0),       # heads of 256, pages that tiles straddle
    (513, 2, 1, 64, 16, 3001, None, 0),       # more sequences than shares take
    (300, 4, 1, 128, 1, 2500, 700, 5),        # windows
    (40, 32, 2, 128, 64, 6000, None, 0)])     # two tiles of heads
def test_ways_that_are_chosen_by_sizes(bits, dtype, B, Hq, Hkv, D, page, most, window, sinks):
    """Ragged sequences of a cache whose pages they share, some of them empty; two calls give the same bits."""
    g = torch.Generator().manual_seed(B + D)
    x = [(torch.randn(most, Hkv, D, generator=g) * torch.where(torch.rand(Hkv, D, generator=g) < 0.05, 6.0, 1.0)).to(dtype) for _ in range(2)]
    cache, table = _cache(*x, bits, page)
    table = torch.stack([table[0][torch.randperm(table.shape[1], generator=g)] for _ in range(B)])
    lens = [most] if B == 1 else [most * (i + 1) // B if i % 9 else 0 for i in torch.randperm(B, generator=g).tolist()]
    few = list(range(B)) if B <= 3 else [0, 1, B // 2, B - 2, B - 1] + [lens.index(max(lens)), lens.index(0)]
    q = torch.randn(B, Hq, D, generator=g).to(dtype)
    gpu = q.cuda(), tdist.QuantizedKVCache(*(t.cuda() for t in cache)), torch.tensor(lens, dtype=torch.int32).cuda(), table.cuda()
    got = [tdist.gqa_fwd_quantized_decode(*gpu, window=window, sinks=sinks).cpu() for _ in range(2)]
    assert torch.equal(*got)
    _compare(got[0][few], q[few], cache, table[few], [lens[b] for b in few], window=window, sinks=sinks)


def test_two_threads_at_once():
    """Calls of the same sizes, each thread on a stream of its own."""
    import threading
    x, w = torch.randn(600, 1024, device="cuda").bfloat16(), torch.randn(2048, 1024, device="cuda")
    k = torch.randn(300, 2, 128, device="cuda").bfloat16()
    q, lens, table = torch.randn(2, 8, 128, device="cuda").bfloat16(), torch.tensor([300, 150]).cuda(), torch.arange(38, device="cuda").view(2, 19)
    torch.cuda.synchronize()

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            cache = tdist.create_quantized_kv_cache(38, 16, 2, 128, 4)
            tdist.kv_cache_write(cache, k, k, torch.arange(300, device="cuda"))
            a, b = tdist.quantize_int8_rowwise(x), tdist.quantize_int8_rowwise(w)
            out = [tdist.gemm_int8(*a, *b) for _ in range(20)] + [tdist.gqa_fwd_quantized_decode(q, cache, lens, table) for _ in range(20)]
            torch.cuda.current_stream().synchronize()
            return out

    got = [None] * 4
    threads = [threading.Thread(target=lambda i=i: got.__setitem__(i, work())) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for out in got:
        assert all(torch.equal(a, b) for a, b in zip(out, got[0]))
        assert all(torch.equal(out[i], out[0]) for i in range(20)) and all(torch.equal(out[i], out[20]) for i in range(20, 40))
