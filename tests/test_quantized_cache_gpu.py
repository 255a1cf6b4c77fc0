"""A KV cache in 8 and 4 bits: writing and reading bit for bit against the plain statement, attention over it against 64 bits.

Bound of the attention, per element, with A = sum_j p_j |v_j| / sum_j p_j, vmax the largest |v| and n keys (all in 64 bits):
* the result's rounding: half a step of its type, 2^-8 (bf16) or 2^-11 (fp16) of itself
* a weight times its value's scale is rounded to fp16: 2^-11 of itself, or 2^-25 of a unit that is at most four times the largest scale
  (the next power of two above it, reached when the largest comes last): n 2^-23 vmax / sum p
* a score is a sum of D / 16 fp32 steps that may truncate (2^-23 of the sum of |q_d k_d| scale each) and a few roundings of its own size, and its
  exponential is good to 2^-21: both move weights and their sum, so twice. The query is brought to 16 bits, rint(q 32512 / max |q|), which is off by
  half a step, max |q| / 65024 < 2^-15.98 max |q|, in each dimension: that times the sum of |k_d| scale is a score's share. The same for 4 bits with |step c| + |least| in the place of |k_d|.
"""
import math

import pytest
import torch

import triton_distributed_b200 as tdist
from triton_distributed_b200.ops import quantized_cache as QC

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _fill(blocks, page, Hkv, D, bits, dtype=torch.bfloat16, seed=0, scale=1.0):
    """A cache on the GPU whose every place is written, by the plain statement on the CPU."""
    g = torch.Generator().manual_seed(seed)
    cache = tdist.create_quantized_kv_cache(blocks, page, Hkv, D, bits, "cpu")
    x = [(torch.randn(blocks * page, Hkv, D, generator=g) * scale * torch.where(torch.rand(Hkv, D, generator=g) < 0.05, 6.0, 1.0)).to(dtype) for _ in range(2)]
    tdist.kv_cache_write(cache, *x, torch.arange(blocks * page))
    return cache, tdist.QuantizedKVCache(*(t.cuda() for t in cache))


def _values64(cache, i):
    """[blocks, page, Hkv, D] in 64 bits, and |step c| + |least| of every value."""
    c, s = cache[i], cache[2 + i].double().transpose(1, 2)
    if cache.bits == 8:
        v = (c.double() - 128.0) * s.unsqueeze(-1)
        return v, v.abs()
    c = torch.stack([c & 15, c >> 4], -1).flatten(-2).double().unflatten(-1, (-1, 64))
    return (c * s[..., 0:1] + s[..., 1:2]).flatten(-2), (c * s[..., 0:1].abs() + s[..., 1:2].abs()).flatten(-2)


def _check_decode(q, cache, lens, table, window=None, sinks=0, scale=None, soft_cap=0.0, **kw):
    """The call against 64 bits on the CPU, element by element."""
    gpu = tdist.QuantizedKVCache(*(t.cuda() for t in cache))
    got = tdist.gqa_fwd_quantized_decode(q.cuda(), gpu, torch.tensor(lens, dtype=torch.int32).cuda(), table.cuda(), window, sinks, scale, soft_cap, **kw).cpu()
    assert got.dtype == q.dtype and got.shape == q.shape
    B, Hq, D = q.shape
    Hkv, page = cache.k.shape[2], cache.k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    (k, ka), (v, va) = _values64(cache, 0), _values64(cache, 1)
    for b, n in enumerate(lens):
        n = min(n, table.shape[1] * page)
        lo = 0 if window is None else max(0, n - window)
        at = torch.cat([torch.arange(0, min(sinks, lo)), torch.arange(lo, max(n, 0))])
        if at.numel() == 0:
            assert (got[b] == 0).all()
            continue
        pages, rows = table[b][at // page].long(), at % page
        qq = q[b].double().view(Hkv, Hq // Hkv, D)
        kb, kab, vb, vab = (t[pages, rows].transpose(0, 1) for t in (k, ka, v, va))
        t = qq @ kb.transpose(1, 2) * scale
        size = (qq.abs() @ kab.transpose(1, 2) * abs(scale)).amax(-1, keepdim=True)
        if soft_cap > 0:
            t = soft_cap * torch.tanh(t / soft_cap)
        p = torch.exp(t - t.amax(-1, keepdim=True))
        l = p.sum(-1, keepdim=True)
        ref, A = p @ vb / l, p @ vab / l
        query = 2.0 ** -15.98 * qq.abs().amax(-1, keepdim=True) * kab.sum(-1).amax(-1).view(-1, 1, 1) * abs(scale)
        moved = 2 * (query + (D / 16 + 6) * 2.0 ** -23 * size + (2.0 ** -20 * soft_cap if soft_cap > 0 else 0.0) + 2.0 ** -20)
        tol = HALF[q.dtype] * ref.abs() + (2.0 ** -11 + moved) * 1.01 * A + at.numel() * 2.0 ** -23 * vab.amax() / l + 2.0 ** -24
        err = (got[b].double().view(Hkv, -1, D) - ref).abs()
        assert bool((err <= tol).all()), (b, n, float(err.max()), float((err / tol).max()))
    return got


def _table(B, blocks_per, spare=1, seed=1):
    order = torch.randperm(B * blocks_per + spare, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    return order[:B * blocks_per].view(B, blocks_per), B * blocks_per + spare


# ---------------------------------------------------------------------------- writing
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("D,Hkv,page,T,dtype", [(128, 8, 16, 33, torch.bfloat16), (64, 3, 1, 1, torch.float16), (256, 1, 5, 200, torch.float16), (128, 12, 64, 1000, torch.bfloat16)])
def test_write_is_the_statement_bit_for_bit(bits, D, Hkv, page, T, dtype):
    blocks = -(-T // page) + 3
    g = torch.Generator().manual_seed(T)
    qkv = (torch.randn(T, 3 * Hkv, D, generator=g) * torch.exp(torch.randn(T, 3 * Hkv, 1, generator=g))).to(dtype)
    qkv[T // 2, Hkv] = 0.0                       # a row of zeros
    qkv[0, -1] = 2.5                             # one value throughout
    slots = torch.randperm(blocks * page, generator=g)[:T].to(torch.int32)
    cpu, gpu = _fill(blocks, page, Hkv, D, bits)
    if T > 4:
        slots[3], slots[4] = -1, blocks * page   # no places of the cache
    tdist.kv_cache_write(cpu, qkv[:, Hkv:2 * Hkv], qkv[:, 2 * Hkv:], slots)
    dev = qkv.cuda()
    tdist.kv_cache_write(gpu, dev[:, Hkv:2 * Hkv], dev[:, 2 * Hkv:], slots.cuda().long())
    for a, b in zip(cpu, gpu):
        assert torch.equal(a, b.cpu())           # what the slots do not name too


@pytest.mark.parametrize("bits", [8, 4])
def test_write_of_extreme_rows(bits):
    """Subnormal, huge, infinite and NaN values; the codes of a bad row are numbers and its scale is NaN."""
    x = torch.randn(12, 1, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    x[1] *= 2.0 ** -110
    x[2] = x[2] * 2.0 ** 120
    x[3, 0, 7] = math.inf
    x[4, 0, 0] = -math.inf
    x[5, 0, 63] = math.nan
    x[6] = x[6].abs() + 1000
    x[7] = -x[7].abs() - 1000
    x[8] = 2.0 ** -133
    x[9, 0, ::2], x[9, 0, 1::2] = 3.3e38, -3.3e38   # a range beyond fp32
    cpu, gpu = _fill(1, 12, 1, 64, bits)
    slots = torch.arange(12)
    tdist.kv_cache_write(cpu, x, x, slots)
    tdist.kv_cache_write(gpu, x.cuda(), x.cuda(), slots.cuda())
    same = [i for i in range(12) if i not in (3, 4, 5)]
    for a, b in zip(cpu, gpu):
        b = b.cpu()
        rows = 1 if a.dtype == torch.uint8 else 2
        pick = (lambda t, i: t[0, i]) if rows == 1 else (lambda t, i: t[0, 0, i])
        for i in same:
            assert torch.equal(pick(a, i).view(torch.uint8 if rows == 1 else torch.int32 if a.dtype == torch.float32 else torch.int16),
                               pick(b, i).view(torch.uint8 if rows == 1 else torch.int32 if a.dtype == torch.float32 else torch.int16)) or (i == 9 and bits == 4), i
        if rows == 2:
            for i in (3, 4, 5):
                assert pick(b, i).isnan().all()


# ---------------------------------------------------------------------------- reading
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("D,Hkv,page,lens,dtype", [(128, 8, 16, [1, 16, 0, 37], torch.bfloat16), (64, 1, 1, [5], torch.float16), (256, 3, 7, [50, 1, 99], torch.float16),
                                                   (128, 8, 64, [3000, 1, 0, 0, 2049], torch.bfloat16)])
def test_read_is_the_statement_bit_for_bit(bits, D, Hkv, page, lens, dtype):
    B = len(lens)
    table, blocks = _table(B, -(-max(lens) // page))
    cpu, gpu = _fill(blocks, page, Hkv, D, bits)
    starts = torch.tensor([3] + [0] * B, dtype=torch.int32)      # three rows before the first, gaps of two, five behind the last
    for b, n in enumerate(lens):
        starts[b + 1] = starts[b] + n + 2
    rows = int(starts[-1]) + 5
    want = tdist.kv_cache_read(cpu, starts, torch.tensor(lens), table, rows, dtype)
    got = tdist.kv_cache_read(gpu, starts.cuda(), torch.tensor(lens).cuda(), table.cuda(), rows, dtype)
    for a, b in zip(want, got):
        assert torch.equal(a, b.cpu())
    out = tuple(torch.full((rows, Hkv, D), 7.0, dtype=dtype, device="cuda") for _ in range(2))
    again = tdist.kv_cache_read(gpu, starts.cuda(), torch.tensor(lens).cuda(), table.cuda(), rows, dtype, out=out)
    assert again[0].data_ptr() == out[0].data_ptr() and all(torch.equal(a, b.cpu()) for a, b in zip(want, out))


def test_read_bounds_what_it_touches():
    """Lengths beyond the table and the gap, pages that the cache does not have, rows that no sequence covers."""
    cpu, gpu = _fill(4, 16, 2, 64, 8)
    table = torch.tensor([[0, 99, 2], [-1, 3, 1]], dtype=torch.int32)
    lens, starts = torch.tensor([1000, 40]), torch.tensor([0, 48, 78])
    want = tdist.kv_cache_read(cpu, starts, lens, table, 90)
    got = tdist.kv_cache_read(gpu, starts.cuda(), lens.cuda(), table.cuda(), 90)
    for a, b in zip(want, got):
        assert torch.equal(a, b.cpu())
    assert (got[0][16:32] == 0).all() and (got[0][78:] == 0).all() and (got[0][64:78] != 0).any()


# ---------------------------------------------------------------------------- attention
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,Hq,Hkv,page,lens", [(128, 32, 8, 16, [1, 15, 16, 17, 700]), (64, 6, 1, 1, [333, 0, 5]), (256, 6, 1, 16, [129]), (128, 16, 1, 5, [64, 1, 257]),
                                                (64, 24, 2, 64, [1000, 3]), (256, 10, 1, 3, [100, 31]), (128, 40, 2, 48, [500])])
def test_decode_against_64_bits(bits, dtype, D, Hq, Hkv, page, lens):
    table, blocks = _table(len(lens), max(1, -(-max(lens) // page)))
    cache, _ = _fill(blocks, page, Hkv, D, bits)
    q = torch.randn(len(lens), Hq, D, generator=torch.Generator().manual_seed(5)).to(dtype)
    _check_decode(q, cache, lens, table)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("splits", [1, 2, 3, 5, 8, 9, 40])
def test_decode_parts_meet(bits, splits):
    """One part, a cluster (odd ones too), a workspace; parts without keys."""
    lens = [1500, 20, 0, 801]
    table, blocks = _table(4, 94)
    cache, _ = _fill(blocks, 16, 2, 128, bits, seed=2)
    q = torch.randn(4, 14, 128, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16)
    _check_decode(q, cache, lens, table, kv_split=splits)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("splits", [0, 1, 2, 40])
@pytest.mark.parametrize("D,Hq,Hkv,page", [(64, 3, 3, 32), (64, 13, 1, 6), (128, 8, 1, 16), (128, 40, 2, 16), (256, 12, 1, 64), (256, 3, 1, 1)])
def test_decode_ways_of_dealing_out(bits, dtype, splits, D, Hq, Hkv, page):
    """Small CTAs, large ones, clusters and shares over the same sequences: ends inside a tile and at its border, none, one past the table."""
    lens = [0, 1, 96, 403, 17, 10 ** 6]
    table, blocks = _table(len(lens), -(-410 // page))
    cache, _ = _fill(blocks, page, Hkv, D, bits, seed=12)
    q = torch.randn(len(lens), Hq, D, generator=torch.Generator().manual_seed(13)).to(dtype)
    _check_decode(q, cache, lens, table, kv_split=splits)
    _check_decode(q, cache, lens, table, window=33, sinks=3, kv_split=splits)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("page", [1, 16, 24])
@pytest.mark.parametrize("window,sinks,cap", [(1, 0, 0.0), (17, 4, 30.0), (100, 37, 0.0), (333, 1, 1000.0), (5000, 4, 5.0)])
def test_decode_windows_and_caps(bits, page, window, sinks, cap):
    """Table entries of pages without a visible key are not pages of the cache, and are not read."""
    lens = [1, 40, 450, 999]
    table, blocks = _table(4, -(-999 // page))
    cache, _ = _fill(blocks, page, 2, 128, bits, seed=3)
    q = 3.0 * torch.randn(4, 8, 128, generator=torch.Generator().manual_seed(7))
    for b, n in enumerate(lens):
        seen = torch.zeros(table.shape[1] * page, dtype=torch.bool)
        seen[max(0, n - window):n] = True
        seen[:min(sinks, n)] = True
        table[b][~seen.view(-1, page).any(1)] = 1 << 30
    _check_decode(q.to(torch.float16), cache, lens, torch.where(table == 1 << 30, -7, table), window, sinks, soft_cap=cap)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("q_size,k_size", [(1e-30, 1.0), (1e4, 1e-4), (1.0, 1e-20), (2.0 ** 60, 2.0 ** -60), (0.0, 1.0)])
def test_decode_of_small_and_large_numbers(bits, q_size, k_size):
    """bf16's range: queries and values far outside fp16's."""
    table, blocks = _table(2, 20)
    cache, _ = _fill(blocks, 16, 1, 64, bits, seed=4, scale=k_size)
    q = (torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(8)) * q_size).to(torch.bfloat16)
    _check_decode(q, cache, [300, 5], table)


@pytest.mark.parametrize("bits", [8, 4])
def test_decode_values_of_rising_scale(bits):
    """Values whose scale rises along the sequence by 2^40 (the unit of the weights moves), weights all alike."""
    table, blocks = _table(1, 64)
    cache = tdist.create_quantized_kv_cache(blocks, 16, 1, 64, bits, "cpu")
    g = torch.Generator().manual_seed(9)
    v = (torch.randn(1024, 1, 64, generator=g) * torch.exp2(torch.linspace(-20, 20, 1024)).view(-1, 1, 1)).to(torch.bfloat16)
    k = torch.randn(1024, 1, 64, generator=g).to(torch.bfloat16)
    at = torch.arange(1024)
    for order in (at, at.flip(0)):
        tdist.kv_cache_write(cache, k, v[order], table[0].long()[at // 16] * 16 + at % 16)
        _check_decode(0.1 * torch.randn(1, 8, 64, generator=g).to(torch.bfloat16), cache, [1024], table)


@pytest.mark.parametrize("bits", [8, 4])
def test_decode_passes_on_nan_and_ignores_what_it_does_not_see(bits):
    table, blocks = _table(3, 4)
    cpu, gpu = _fill(blocks, 16, 2, 64, bits, seed=5)
    q = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(10)).to(torch.bfloat16).cuda()
    lens = torch.tensor([50, 50, 50], dtype=torch.int32).cuda()
    clean = tdist.gqa_fwd_quantized_decode(q, gpu, lens, table.cuda())
    bad = torch.full((1, 2, 64), math.nan, dtype=torch.bfloat16, device="cuda")
    ok = torch.ones((1, 2, 64), dtype=torch.bfloat16, device="cuda")
    spot = lambda b, j: (table[b, j // 16] * 16 + j % 16).view(1).cuda()   # noqa: E731
    tdist.kv_cache_write(gpu, bad, bad, spot(0, 50))        # behind the last key, in its page
    tdist.kv_cache_write(gpu, bad, ok, spot(1, 3))          # a key that is seen
    tdist.kv_cache_write(gpu, ok, bad, spot(2, 49))         # a value that is seen
    got = tdist.gqa_fwd_quantized_decode(q, gpu, lens, table.cuda())
    assert torch.equal(got[0], clean[0]) and got[1:].isnan().all()
    # a window that leaves the bad rows out
    got = tdist.gqa_fwd_quantized_decode(q, gpu, lens - 1, table.cuda(), window=20)
    assert not got.isnan().any()


def test_decode_takes_strided_caches_and_given_outputs():
    """Layers of one allocation: the pages of a layer are not contiguous."""
    L, page, Hkv, D = 3, 16, 2, 128
    table, blocks = _table(2, 10)
    codes = torch.zeros(blocks, L, 2, page, Hkv, D, dtype=torch.uint8)
    scales = torch.zeros(blocks, L, 2, Hkv, page)
    cache, _ = _fill(blocks, page, Hkv, D, 8, seed=6)
    codes[:, 1, 0], codes[:, 1, 1], scales[:, 1, 0], scales[:, 1, 1] = cache
    gc, gs = codes.cuda(), scales.cuda()
    view = tdist.QuantizedKVCache(gc[:, 1, 0], gc[:, 1, 1], gs[:, 1, 0], gs[:, 1, 1])
    q = torch.randn(2, 4, D).to(torch.float16).cuda()
    lens = torch.tensor([150, 31]).cuda()
    out = torch.empty_like(q)
    got = tdist.gqa_fwd_quantized_decode(q, view, lens, table.cuda(), out=out)
    want = tdist.gqa_fwd_quantized_decode(q, tdist.QuantizedKVCache(*(t.cuda() for t in cache)), lens, table.cuda())
    assert got.data_ptr() == out.data_ptr() and torch.equal(got, want)
    k = torch.randn(5, Hkv, D).to(torch.float16).cuda()
    tdist.kv_cache_write(view, k, k, torch.tensor([0, 17, 33, 34, 40]).cuda())
    ref = QC.ref_quantize_rows(k.cpu(), 8)
    assert torch.equal(gc[0, 1, 0, 0].cpu(), ref[0][0]) and torch.equal(gs[1, 1, 1, :, 1].cpu(), ref[1][1])
    codes[0, 1, :, 0], codes[1, 1, :, 1], codes[2, 1, :, 1], codes[2, 1, :, 2], codes[2, 1, :, 8] = ref[0]
    assert torch.equal(gc.cpu(), codes)            # the other layers kept their bytes


@pytest.mark.parametrize("bits", [8, 4])
def test_write_decode_and_read_in_a_captured_graph(bits):
    """A step of serving: the token's k and v are written, then attended to with all before; replayed with new tokens."""
    B, Hq, Hkv, D, page = 3, 8, 2, 128, 16
    table, blocks = _table(B, 40)
    cpu, gpu = _fill(blocks, page, Hkv, D, bits, seed=7)
    dt = table.cuda()
    lens = torch.tensor([100, 1, 620], dtype=torch.int32).cuda()
    slots = torch.full((B,), -1, dtype=torch.int32, device="cuda")   # the warm-up writes nothing
    k, v, q = (torch.randn(B, h, D, device="cuda").to(torch.bfloat16) for h in (Hkv, Hkv, Hq))
    starts = torch.tensor([0, 640, 1280, 1920], dtype=torch.int32, device="cuda")

    def step():
        tdist.kv_cache_write(gpu, k, v, slots)
        o = tdist.gqa_fwd_quantized_decode(q, gpu, lens, dt, kv_split=12)
        return o, tdist.kv_cache_read(gpu, starts, lens, dt, 1920)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, (rk, rv) = step()
    for turn in range(3):
        lens.copy_(torch.tensor([100 + turn, 1 + turn, 620 + turn]))
        for t in (k, v, q):
            t.normal_()
        at = (lens - 1).cpu().long()
        slots.copy_(table.gather(1, (at // page).view(-1, 1)).view(-1) * page + at % page)
        graph.replay()
        torch.cuda.synchronize()
        tdist.kv_cache_write(cpu, k.cpu(), v.cpu(), slots.cpu())
        assert all(torch.equal(a, b.cpu()) for a, b in zip(cpu, gpu))
        want = tdist.kv_cache_read(cpu, starts.cpu(), lens.cpu(), table, 1920)
        assert torch.equal(want[0], rk.cpu()) and torch.equal(want[1], rv.cpu())
        _check_decode(q.cpu(), cpu, lens.tolist(), table)
        eager = tdist.gqa_fwd_quantized_decode(q, gpu, lens, dt, kv_split=12)
        assert torch.equal(eager, o)


def test_read_back_as_pages_feeds_the_prefill():
    """A prompt's chunk: written, its sequences read back as a paged cache in bf16, prefill over that."""
    Hq, Hkv, D, page, lens, new = 8, 2, 128, 16, [100, 37], [30, 37]
    table, blocks = _table(2, 7)
    cpu, gpu = _fill(blocks, page, Hkv, D, 8, seed=8)
    k, v = (torch.randn(sum(new), Hkv, D, device="cuda").to(torch.bfloat16) for _ in range(2))
    q = torch.randn(sum(new), Hq, D, device="cuda").to(torch.bfloat16)
    at = [torch.arange(n - t, n) for n, t in zip(lens, new)]
    slots = torch.cat([table[b].long()[a // page] * page + a % page for b, a in enumerate(at)])
    tdist.kv_cache_write(gpu, k, v, slots.cuda())
    tdist.kv_cache_write(cpu, k.cpu(), v.cpu(), slots)
    each = 7 * page
    starts = torch.tensor([0, each, 2 * each], dtype=torch.int32).cuda()
    kl = torch.tensor(lens, dtype=torch.int32).cuda()
    rk, rv = tdist.kv_cache_read(gpu, starts, kl, table.cuda(), 2 * each)
    pages = torch.arange(14, dtype=torch.int32, device="cuda").view(2, 7)
    qs = torch.tensor([0, new[0], sum(new)], dtype=torch.int32).cuda()
    got = tdist.gqa_fwd_window_prefill(q, rk.view(14, page, Hkv, D), rv.view(14, page, Hkv, D), qs, kl, pages)
    for b, n in enumerate(lens):
        kk, vv = (t[b * each:b * each + n].double() for t in (rk, rv))
        qq = q[int(qs[b]):int(qs[b + 1])].double().view(new[b], Hkv, Hq // Hkv, D)
        s = torch.einsum("nhgd,khd->hgnk", qq, kk) * D ** -0.5
        pos = torch.arange(n - new[b], n, device="cuda").view(-1, 1)
        s = s.masked_fill(torch.arange(n, device="cuda").view(1, -1) > pos, -math.inf)
        p = torch.softmax(s, -1)
        ref = torch.einsum("hgnk,khd->nhgd", p, vv).reshape(new[b], Hq, D)
        size = torch.einsum("hgnk,khd->nhgd", p, vv.abs()).reshape(new[b], Hq, D)
        # weights and the result are rounded to bf16, scores off by fp32 sums
        tol = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -14) * size
        assert bool(((got[int(qs[b]):int(qs[b + 1])].double() - ref).abs() <= tol).all())


def test_two_streams_at_once():
    table, blocks = _table(4, 30)
    cpu, gpu = _fill(blocks, 16, 2, 128, 8, seed=9)
    q = torch.randn(4, 8, 128, generator=torch.Generator().manual_seed(12)).to(torch.bfloat16).cuda()
    lens, dt = torch.tensor([480, 10, 300, 77], dtype=torch.int32).cuda(), table.cuda()
    want = {s: tdist.gqa_fwd_quantized_decode(q, gpu, lens, dt, kv_split=s) for s in (1, 4, 20)}
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(30):
        with torch.cuda.stream(streams[i % 2]):
            got.append(((1, 4, 20)[i % 3], tdist.gqa_fwd_quantized_decode(q, gpu, lens, dt, kv_split=(1, 4, 20)[i % 3])))
    torch.cuda.synchronize()
    assert all(torch.equal(want[s], o) for s, o in got)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("D,page,splits", [(128, 16, 1), (128, 16, 2), (64, 16, 1), (256, 16, 1), (128, 5, 1)])
def test_decode_goes_round_its_rings_often(bits, D, page, splits):
    """Many tiles per warp, whose loads land in any order, on a full machine: the same result every time, and the right one."""
    B, Hkv, n = 40, 4, 6000
    table, blocks = _table(1, -(-n // page))
    cpu, gpu = _fill(blocks, page, Hkv, D, bits, seed=11)
    q = torch.randn(B, 8, D, generator=torch.Generator().manual_seed(13)).to(torch.float16)
    lens = torch.tensor([n - 16 * b for b in range(B)], dtype=torch.int32)
    args = q.cuda(), gpu, lens.cuda(), table.expand(B, -1).cuda()
    got = [tdist.gqa_fwd_quantized_decode(*args, kv_split=splits) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(got[0], o) for o in got)
    one = _check_decode(q[-1:], cpu, [int(lens[-1])], table, kv_split=splits)
    assert torch.equal(one[0], got[0][-1].cpu())
