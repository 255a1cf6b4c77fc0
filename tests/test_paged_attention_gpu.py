"""Windowed decode and prefill and shared-prefix decode against plain statements in 64 bits.

Bounds: u is half a unit of the 16-bit type's last place (2^-8 of a value for bf16 with its 8 significant bits, 2^-11 for fp16, the largest relative
rounding error). P is rounded once (u of sum p |v|) and the result once (u of it); S, O and the sums are fp32 (2^-24 each step, over at
most some hundred steps of a block and as many blocks: 1e-4 of sum p |v| covers it with the exponential's 2^-22 and the scores' error of
2^-24 x sum |q k| scale, a few tens here). A soft cap adds its fp32 evaluation, 2^-21 of the cap, twice (its own score's, the sum's)."""
import math

import pytest
import torch

import triton_distributed_b200 as tdist
from triton_distributed_b200 import _lib
from triton_distributed_b200.runtime import check_status

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": (torch.bfloat16, 2.0 ** -8), "fp16": (torch.float16, 2.0 ** -11)}


def _exact(q, k, v, seen, scale, cap):
    """float64: q [n, Hq, D], k, v [keys, Hkv, D], seen [n, keys] -> out, sum p |v|."""
    n, Hq, D = q.shape
    Hkv = k.shape[1]
    s = torch.einsum("nhgd,khd->hgnk", q.double().view(n, Hkv, Hq // Hkv, D), k.double()) * scale
    if cap > 0:
        s = cap * torch.tanh(s / cap)
    s = s.masked_fill(~seen, float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == float("-inf"), 0.0, m))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    out = torch.einsum("hgnk,khd->nhgd", p, v.double()).reshape(n, Hq, D)
    return out, torch.einsum("hgnk,khd->nhgd", p, v.double().abs()).reshape(n, Hq, D)


def _mask(n, kv, window, sinks, dev):
    pos, j = torch.arange(kv - n, kv, device=dev).unsqueeze(1), torch.arange(kv, device=dev)
    seen = j <= pos
    if window is not None:
        seen = seen & ((j > pos - window) | (j < sinks))
    return seen


def _cache(pages, page, Hkv, D, dt, dev):
    return torch.randn(pages, page, Hkv, D, device=dev).to(dt), torch.randn(pages, page, Hkv, D, device=dev).to(dt)


def _keys(cache, table, n):
    return cache[table.long()].flatten(0, 1)[:n]


def _compare(out, ref, spread, u, cap=0.0):
    bound = u * (spread + ref.abs()) + (1e-4 + 2 * cap * 2.0 ** -21) * spread + 1e-6
    worst = ((out.double() - ref).abs() - bound).max()
    assert torch.isfinite(out).all() and worst <= 0, float(worst)


def _prefill_case(dev, dtype, Hq, Hkv, D, page, lens, window, sinks, cap=0.0, scale=None, poison=True, kv_split=-1, fused=False):
    """lens: (query tokens, keys) per sequence. Pages without a visible key are out of the table, cache rows behind a
    sequence's last key are NaN."""
    dt, u = DTYPES[dtype]
    torch.manual_seed(sum(n + 3 * kv for n, kv in lens) + D + page)
    B, most = len(lens), max(1, max(-(-kv // page) for _, kv in lens))
    k, v = _cache(B * most + 2, page, Hkv, D, dt, dev)
    table = torch.randperm(B * most + 2, device=dev)[:B * most].view(B, most).to(torch.int32)
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    q = torch.randn(starts[-1], Hq + (2 * Hkv if fused else 0), D, device=dev).to(dt)[:, :Hq]
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    refs, spreads = [], []
    for b, (n, kv) in enumerate(lens):
        if n == 0:
            continue
        if kv == 0:
            refs.append(torch.zeros(n, Hq, D, dtype=torch.float64, device=dev))
            spreads.append(refs[-1])
            continue
        seen = _mask(n, kv, window, sinks, dev)
        r, s = _exact(q[starts[b]:starts[b + 1]], _keys(k, table[b], kv), _keys(v, table[b], kv), seen, scale, cap)
        refs.append(r)
        spreads.append(s)
        if poison:
            pages = seen.any(0)
            for i in range(most):
                part = pages[i * page:(i + 1) * page]
                if not bool(part.any()):
                    table[b, i] = 0x3FFFFFFF   # given back: never read
                elif (i + 1) * page > kv:
                    k[int(table[b, i]), kv - i * page:] = float("nan")
                    v[int(table[b, i]), kv - i * page:] = float("nan")
    out = tdist.gqa_fwd_window_prefill(q, k, v, torch.tensor(starts, dtype=torch.int32, device=dev),
                                       torch.tensor([kv for _, kv in lens], dtype=torch.int32, device=dev), table, window=window,
                                       sinks=sinks, scale=scale, soft_cap=cap, kv_split=kv_split)
    check_status()
    _compare(out, torch.cat(refs), torch.cat(spreads), u, cap)
    return out


@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 2), (16, 2), (6, 1), (24, 2), (5, 1)])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 16), (256, 64), (128, 1), (64, 3)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_prefill_heads_pages_types(cuda_device, Hq, Hkv, D, page, dtype):
    _prefill_case(cuda_device, dtype, Hq, Hkv, D, page, [(1, 1), (33, 33), (5, 300), (70, 131), (128, 128)], 40, 4)


@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (1, 1), (17, 3), (127, 4), (128, 0), (129, 130), (1000, 5000)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_prefill_windows(cuda_device, window, sinks, D):
    lens = [(1, 1000), (2, 2), (127, 127), (129, 700), (300, 300), (64, 1024), (257, 513)]
    _prefill_case(cuda_device, "bf16", 8, 2, D, 16, lens, window, sinks)
    _prefill_case(cuda_device, "fp16", 3, 3, D, 16, lens, window, sinks, fused=True)


@pytest.mark.parametrize("splits", [1, 2, 5, 16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_prefill_splits(cuda_device, splits, D):
    for lens in ([(3, 2500)], [(200, 1500), (1, 9)]):
        _prefill_case(cuda_device, "bf16", 8, 2, D, 16, lens, None, 0, kv_split=splits)
        _prefill_case(cuda_device, "bf16", 8, 2, D, 16, lens, 700, 5, kv_split=splits)


@pytest.mark.parametrize("scale", [0.3, -0.2, 0.0])
@pytest.mark.parametrize("cap", [0.0, 15.0])
def test_prefill_scale_and_cap(cuda_device, scale, cap):
    _prefill_case(cuda_device, "bf16", 4, 1, 128, 16, [(150, 400)], 200, 2, cap=cap, scale=scale)


def test_prefill_rows_that_see_nothing(cuda_device):
    # no keys, more query tokens than keys (their positions lie before the first key), sequences without tokens
    out = _prefill_case(cuda_device, "bf16", 8, 2, 128, 16, [(4, 0), (0, 50), (10, 3), (0, 0), (40, 40)], 8, 2)
    assert (out[:4] == 0).all() and (out[4:11] == 0).all() and (out[11:14] != 0).any()


def test_prefill_long_context_offsets(cuda_device):
    """Cache rows beyond 2^31 elements; a chunk at the end of a long context."""
    dev, D, page, Hkv, kv = cuda_device, 128, 64, 8, 3000
    need = -(-kv // page)
    pages = (1 << 31) // (page * Hkv * D) + need + 1
    if torch.cuda.get_device_properties(dev).total_memory < 24 << 30:
        pytest.skip("needs 9 GB for the caches")
    k = torch.zeros(pages, page, Hkv, D, dtype=torch.bfloat16, device=dev)
    v = torch.zeros_like(k)
    table = torch.arange(pages - need, pages, dtype=torch.int32, device=dev).view(1, need)
    k[pages - need:].normal_()
    v[pages - need:].normal_()
    q = torch.randn(70, 16, D, device=dev).to(torch.bfloat16)
    out = tdist.gqa_fwd_window_prefill(q, k, v, torch.tensor([0, 70], device=dev), torch.tensor([kv], device=dev), table, window=2000, sinks=4)
    dec = tdist.gqa_fwd_window_decode(q[69:].contiguous(), k, v, torch.tensor([kv], device=dev), table, window=2000, sinks=4)
    check_status()
    ref, spread = _exact(q, _keys(k, table[0], kv), _keys(v, table[0], kv), _mask(70, kv, 2000, 4, dev), D ** -0.5, 0.0)
    _compare(out, ref, spread, 2.0 ** -8)
    _compare(dec, ref[69:], spread[69:], 2.0 ** -8)


@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 2), (32, 2), (6, 1)])
@pytest.mark.parametrize("D,page", [(64, 16), (64, 1), (128, 16), (128, 3), (256, 64)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (16, 1), (100, 4), (513, 37)])
@pytest.mark.parametrize("dtype,cap", [("bf16", 0.0), ("fp16", 12.0)])
def test_window_decode(cuda_device, Hq, Hkv, D, page, window, sinks, dtype, cap):
    dev, (dt, u) = cuda_device, DTYPES[dtype]
    torch.manual_seed(Hq + D + page + sinks)
    lens = [0, 1, 2, 15, 16, 17, 99, 100, 101, 513, 900, 3000]
    B, most = len(lens), -(-max(lens) // page)
    k, v = _cache(B * most, page, Hkv, D, dt, dev)
    table = torch.randperm(B * most, device=dev).view(B, most).to(torch.int32)
    q = torch.randn(B, Hq, D, device=dev).to(dt)
    refs = [_exact(q[b:b + 1], _keys(k, table[b], n), _keys(v, table[b], n), _mask(1, n, window, sinks, dev), 0.15, cap) if n else
            (torch.zeros(1, Hq, D, dtype=torch.float64, device=dev),) * 2 for b, n in enumerate(lens)]
    for b, n in enumerate(lens):
        for i in range(most):
            seen = [j for j in range(i * page, min(n, (i + 1) * page)) if window is None or j >= n - window or j < sinks]
            if not seen:
                table[b, i] = int(table[b, -1]) if n > 0 else 0   # a page in use elsewhere: its keys must not count
    tl = torch.tensor(lens, dtype=torch.int32, device=dev)
    for splits in (-1, 1, 3, 16):
        out = tdist.gqa_fwd_window_decode(q, k, v, tl, table, window=window, sinks=sinks, scale=0.15, soft_cap=cap, kv_split=splits)
        check_status()
        _compare(out, torch.cat([r for r, _ in refs]), torch.cat([s for _, s in refs]), u, cap)
        assert (out[0] == 0).all()


def _prefix_case(dev, dtype, B, Hq, Hkv, D, page, prefix, lens, cap=0.0, scale=None, kv_split=-1, as_number=False):
    dt, u = DTYPES[dtype]
    torch.manual_seed(B + Hq + D + prefix)
    own, pre = max(1, -(-max(lens) // page)), -(-prefix // page)
    k, v = _cache(B * own + pre + 1, page, Hkv, D, dt, dev)
    order = torch.randperm(B * own + pre + 1, device=dev).to(torch.int32)
    table, ptable = order[:B * own].view(B, own), order[B * own:B * own + pre]
    q = torch.randn(B, Hq, D, device=dev).to(dt)
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    refs = []
    for b, n in enumerate(lens):
        kk = torch.cat([_keys(k, ptable, prefix), _keys(k, table[b], n)])
        vv = torch.cat([_keys(v, ptable, prefix), _keys(v, table[b], n)])
        seen = torch.ones(1, prefix + n, dtype=torch.bool, device=dev)
        refs.append(_exact(q[b:b + 1], kk, vv, seen, scale, cap) if prefix + n else (torch.zeros(1, Hq, D, dtype=torch.float64, device=dev),) * 2)
    if pre and prefix % page:
        k[int(ptable[-1]), prefix % page:] = float("nan")
        v[int(ptable[-1]), prefix % page:] = float("nan")
    length = prefix if as_number else torch.tensor([prefix], dtype=torch.int32, device=dev)
    out = tdist.gqa_fwd_shared_prefix_decode(q, k, v, length, ptable, torch.tensor(lens, dtype=torch.int32, device=dev), table, scale=scale,
                                             soft_cap=cap, kv_split=kv_split)
    check_status()
    _compare(out, torch.cat([r for r, _ in refs]), torch.cat([s for _, s in refs]), u, cap)


@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 2), (32, 2), (6, 1), (24, 2)])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 16), (128, 1), (256, 64), (64, 5)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_shared_prefix(cuda_device, Hq, Hkv, D, page, dtype):
    _prefix_case(cuda_device, dtype, 5, Hq, Hkv, D, page, 333, [1, 0, 17, 200, 64])
    _prefix_case(cuda_device, dtype, 67, Hq, Hkv, D, page, 700, [(7 * i) % 90 for i in range(67)])


@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 127, 128, 129, 2049])
@pytest.mark.parametrize("B", [1, 32, 33, 130])
def test_shared_prefix_lengths(cuda_device, prefix, B):
    _prefix_case(cuda_device, "bf16", B, 8, 2, 128, 16, prefix, [(5 * i) % 40 for i in range(B)], as_number=prefix == 127)


@pytest.mark.parametrize("splits", [1, 2, 7, 64])
@pytest.mark.parametrize("cap,scale", [(0.0, None), (20.0, 0.4)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_shared_prefix_splits(cuda_device, splits, cap, scale, D):
    _prefix_case(cuda_device, "bf16", 9, 8, 2, D, 16, 3001, [300] * 9, cap=cap, scale=scale, kv_split=splits)
    _prefix_case(cuda_device, "fp16", 70, 8, 2, D, 16, 1500, [3] * 70, cap=cap, scale=scale, kv_split=splits)


def test_interleaved_caches_and_out(cuda_device):
    """k and v as halves of one cache, indices in 64 bits, the result into a given tensor, on a stream of its own."""
    dev = cuda_device
    torch.manual_seed(3)
    kv = torch.randn(40, 2, 16, 2, 128, device=dev).to(torch.bfloat16)
    k, v = kv[:, 0], kv[:, 1]
    table = torch.randperm(40, device=dev).view(2, 20)
    q = torch.randn(100, 8, 128, device=dev).to(torch.bfloat16)
    out = torch.empty_like(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = tdist.gqa_fwd_window_prefill(q, k, v, torch.tensor([0, 60, 100], device=dev), torch.tensor([300, 200], device=dev), table,
                                           window=90, sinks=2, out=out)
    s.synchronize()
    check_status()
    assert got is out
    for b, (a, e, n) in enumerate(((0, 60, 300), (60, 100, 200))):
        r, sp = _exact(q[a:e], _keys(k, table[b], n), _keys(v, table[b], n), _mask(e - a, n, 90, 2, dev), 128 ** -0.5, 0.0)
        _compare(out[a:e], r, sp, 2.0 ** -8)


def test_replays_from_a_graph(cuda_device):
    """Captured once, replayed with other lengths in the same tensors."""
    dev = cuda_device
    torch.manual_seed(4)
    B, page = 6, 16
    k, v = _cache(B * 40 + 30, page, 2, 128, torch.bfloat16, dev)
    table = torch.randperm(B * 40 + 30, device=dev).to(torch.int32)
    own, pre = table[:B * 40].view(B, 40), table[B * 40:]
    q = torch.randn(B, 8, 128, device=dev).to(torch.bfloat16)
    lens, plen = torch.full((B,), 100, dtype=torch.int32, device=dev), torch.tensor([200], dtype=torch.int32, device=dev)
    starts = torch.arange(B + 1, dtype=torch.int32, device=dev)

    def step():
        return (tdist.gqa_fwd_window_decode(q, k, v, lens, own, window=64, sinks=3), tdist.gqa_fwd_window_prefill(q, k, v, starts, lens, own, window=64, sinks=3),
                tdist.gqa_fwd_shared_prefix_decode(q, k, v, plen, pre, lens, own))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step()
    for n, p in ((100, 200), (1, 480), (640, 1), (333, 77)):
        lens.fill_(n)
        plen.fill_(p)
        g.replay()
        torch.cuda.synchronize()
        check_status()
        for a, b in zip(outs, step()):
            assert torch.equal(a, b)
        for b in range(B):
            r, sp = _exact(q[b:b + 1], _keys(k, own[b], n), _keys(v, own[b], n), _mask(1, n, 64, 3, dev), 128 ** -0.5, 0.0)
            _compare(outs[0][b:b + 1], r, sp, 2.0 ** -8)
            _compare(outs[1][b:b + 1], r, sp, 2.0 ** -8)
            kk, vv = torch.cat([_keys(k, pre, p), _keys(k, own[b], n)]), torch.cat([_keys(v, pre, p), _keys(v, own[b], n)])
            r, sp = _exact(q[b:b + 1], kk, vv, torch.ones(1, n + p, dtype=torch.bool, device=dev), 128 ** -0.5, 0.0)
            _compare(outs[2][b:b + 1], r, sp, 2.0 ** -8)


def test_scores_that_rise_and_extremes(cuda_device):
    """Maxima that rise by more than 2^8 from block to block, and fall; infinite scores in one direction are weights of zero."""
    dev = cuda_device
    for sign in (1.0, -1.0):
        n, D = 1024, 128
        q = torch.ones(40, 4, D, device=dev).to(torch.bfloat16)
        k = (torch.linspace(-2, 2, n, device=dev) * sign).view(n, 1, 1).expand(n, 1, D).to(torch.bfloat16).contiguous().view(n // 16, 16, 1, D)
        v = torch.randn(n // 16, 16, 1, D, device=dev).to(torch.bfloat16)
        table = torch.arange(n // 16, dtype=torch.int32, device=dev).view(1, -1)
        args = (torch.tensor([0, 40], device=dev), torch.tensor([n], device=dev), table)
        for split in (1, 2):
            out = tdist.gqa_fwd_window_prefill(q, k, v, *args, scale=1.0, kv_split=split)
            check_status()
            r, sp = _exact(q, k.flatten(0, 1), v.flatten(0, 1), _mask(40, n, None, 0, dev), 1.0, 0.0)
            _compare(out, r, sp, 2.0 ** -8)


def test_refusals(cuda_device):
    dev = cuda_device
    k, v = _cache(8, 16, 2, 128, torch.bfloat16, dev)
    table, lens = torch.zeros(2, 4, dtype=torch.int32, device=dev), torch.ones(2, dtype=torch.int32, device=dev)
    q, starts = torch.zeros(2, 8, 128, dtype=torch.bfloat16, device=dev), torch.arange(3, device=dev)
    pre, plen = torch.zeros(4, dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
    P, W, S = tdist.gqa_fwd_window_prefill, tdist.gqa_fwd_window_decode, tdist.gqa_fwd_shared_prefix_decode
    with pytest.raises(ValueError):
        P(q, k, v, starts, lens, table, window=0)
    with pytest.raises(ValueError):
        W(q, k, v, lens, table, window=4, sinks=-1)
    with pytest.raises(ValueError):
        P(q, k, v, starts[:2], lens, table)
    with pytest.raises(ValueError):
        W(q, k, v, lens[:1], table)
    with pytest.raises(TypeError):
        P(q.float(), k, v, starts, lens, table)
    with pytest.raises(TypeError):
        P(q, k, v, starts.float(), lens, table)
    with pytest.raises(ValueError):
        P(q[..., :96], k[..., :96], v[..., :96], starts, lens, table)
    with pytest.raises(ValueError):
        P(q[:, :7], k, v, starts, lens, table)
    with pytest.raises(ValueError):
        P(q, k, v[:4], starts, lens, table)
    with pytest.raises(ValueError):
        P(q, k, v, starts.cpu(), lens, table)
    with pytest.raises(ValueError):
        P(q, k, v, starts, lens, table, soft_cap=float("nan"))
    with pytest.raises(ValueError):
        S(q.transpose(0, 1).contiguous().transpose(0, 1), k, v, plen, pre, lens, table)
    with pytest.raises(ValueError):
        S(q, k, v, lens, pre, lens, table)
    with pytest.raises(ValueError):
        P(q, k, v, starts, lens, table, out=torch.empty(2, 8, 128, device=dev))
    odd = torch.zeros(2 * 8 * 129, dtype=torch.bfloat16, device=dev).view(2, 8, 129)[..., :128]
    with pytest.raises(_lib.TdistError):
        P(odd, k, v, starts, lens, table)
    assert P(q[:0], k, v, torch.zeros(3, dtype=torch.int32, device=dev), lens, table).shape == (0, 8, 128)


def test_more_tokens_than_keys_without_a_window(cuda_device):
    """The first query positions lie before the first key: they see nothing, the later ones what is there."""
    for lens in ([(40, 7)], [(300, 200), (5, 1), (70, 64)]):
        out = _prefill_case(cuda_device, "bf16", 8, 2, 128, 16, lens, None, 0)
        assert (out[:lens[0][0] - lens[0][1]] == 0).all() and (out[lens[0][0] - lens[0][1]:lens[0][0]] != 0).any()
        _prefill_case(cuda_device, "fp16", 8, 2, 64, 16, lens, None, 3)


@pytest.mark.parametrize("page", [16, 1])
def test_caches_with_heads_before_tokens(cuda_device, page):
    """[blocks, Hkv, page, D] in memory, seen as [blocks, page, Hkv, D]; a cache of more heads than are used."""
    dev = cuda_device
    torch.manual_seed(page)
    for D in (64, 128, 256):
        base = torch.randn(2, 40 * 16 // page, 6, page, D, device=dev).to(torch.bfloat16)
        k, v = (base[i].permute(0, 2, 1, 3)[:, :, 1:4] for i in range(2))
        need = -(-300 // page)
        order = torch.randperm(k.shape[0], device=dev).to(torch.int32)
        table = order[:2 * need].view(2, need)
        q = torch.randn(90, 12, D, device=dev).to(torch.bfloat16)
        lens = torch.tensor([300, 77], dtype=torch.int32, device=dev)
        out = tdist.gqa_fwd_window_prefill(q, k, v, torch.tensor([0, 60, 90], device=dev), lens, table, window=120, sinks=3)
        dec = tdist.gqa_fwd_window_decode(q[[59, 89]].contiguous(), k, v, lens, table, window=120, sinks=3)
        pre = tdist.gqa_fwd_shared_prefix_decode(q[:2].contiguous(), k, v, 200, table[0], torch.tensor([77, 0], device=dev), table.flip(0))
        check_status()
        for b, (a, e, n) in enumerate(((0, 60, 300), (60, 90, 77))):
            r, sp = _exact(q[a:e], _keys(k, table[b], n), _keys(v, table[b], n), _mask(e - a, n, 120, 3, dev), D ** -0.5, 0.0)
            _compare(out[a:e], r, sp, 2.0 ** -8)
            _compare(dec[b:b + 1], r[-1:], sp[-1:], 2.0 ** -8)
            kk = torch.cat([_keys(k, table[0], 200), _keys(k, table[1], 77)]) if b == 0 else _keys(k, table[0], 200)
            vv = torch.cat([_keys(v, table[0], 200), _keys(v, table[1], 77)]) if b == 0 else _keys(v, table[0], 200)
            r, sp = _exact(q[b:b + 1], kk, vv, torch.ones(1, kk.shape[0], dtype=torch.bool, device=dev), D ** -0.5, 0.0)
            _compare(pre[b:b + 1], r, sp, 2.0 ** -8)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_soft_caps_on_both_sides_of_the_polynomial(cuda_device, D):
    """Scores far below the cap, around it, and beyond it, in one batch."""
    dev = cuda_device
    for scale, cap in ((0.01, 30.0), (0.3, 2.0), (2.0, 5.0)):
        _prefill_case(dev, "fp16", 8, 2, D, 16, [(40, 400), (70, 90)], 300, 2, cap=cap, scale=scale)


def test_refusals_of_head_counts_and_parts(cuda_device):
    dev = cuda_device
    k, v = _cache(8, 16, 1, 128, torch.bfloat16, dev)
    table, lens, pre = torch.zeros(2, 4, dtype=torch.int32, device=dev), torch.ones(2, dtype=torch.int32, device=dev), torch.zeros(4, dtype=torch.int32, device=dev)
    q = torch.zeros(2, 17, 128, dtype=torch.bfloat16, device=dev)
    with pytest.raises(ValueError):
        tdist.gqa_fwd_window_decode(q, k, v, lens, table, window=4)
    with pytest.raises(ValueError):
        tdist.gqa_fwd_shared_prefix_decode(q, k, v, 5, pre, lens, table)
    with pytest.raises(ValueError):
        tdist.gqa_fwd_shared_prefix_decode(q[:, :8].contiguous(), k, v, 5, pre, lens, table, kv_split=201)
    assert tdist.gqa_fwd_window_prefill(q, k, v, torch.arange(3, device=dev), lens, table, window=4).shape == q.shape   # prefill takes them


@pytest.mark.parametrize("indices", [torch.int32, torch.int64])
def test_shared_prefix_behind_writes_of_its_inputs(cuda_device, indices):
    """Calls one after the other without a wait between them, each behind kernels that write its queries, caches, table and lengths: the own
    keys' kernel starts while the prefix' one runs, but not before what both read is there. Integers in 64 bits are converted on the way."""
    dev, B, P, page = cuda_device, 70, 4096, 16
    torch.manual_seed(8)
    pages, most = P // page + B * 8, 8
    rounds = []
    for _ in range(4):
        k, v = _cache(pages, page, 2, 128, torch.bfloat16, dev)
        order = torch.randperm(pages, device=dev)
        rounds.append((torch.randn(B, 8, 128, device=dev).to(torch.bfloat16), k, v, torch.tensor([P - 7], device=dev).to(indices),
                       order[:P // page].to(indices), torch.randint(0, most * page + 1, (B,), device=dev).to(indices),
                       order[P // page:].view(B, most).to(indices)))
    now = [torch.zeros_like(t) for t in rounds[0]]
    outs = []
    for given in rounds * 3:
        for dst, src in zip(now, given):
            dst.copy_(src)
        outs.append(tdist.gqa_fwd_shared_prefix_decode(*now))
    check_status()
    for i, (q, k, v, n, first, lens, table) in enumerate(rounds):
        for out in outs[i + 4::4]:
            assert torch.equal(out, outs[i])
        for b in range(0, B, 9):
            own = int(lens[b])
            keys = [torch.cat([_keys(c, first, int(n)), _keys(c, table[b], own)]) for c in (k, v)]
            r, s = _exact(q[b:b + 1], keys[0], keys[1], torch.ones(1, int(n) + own, dtype=torch.bool, device=dev), 128 ** -0.5, 0.0)
            _compare(outs[i][b:b + 1], r, s, 2.0 ** -8)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_many_short_rows(cuda_device, D):
    """Tiles of one to four blocks of keys, thousands of them one after the other: every wait ends, every call gives the same."""
    dev, n = cuda_device, 6000
    torch.manual_seed(9)
    k, v = _cache(n // 16 + 1, 16, 4, D, torch.bfloat16, dev)
    q = torch.randn(n, 8, D, device=dev).to(torch.bfloat16)
    table = torch.randperm(n // 16 + 1, device=dev).view(1, -1).to(torch.int32)
    starts, lens = torch.tensor([0, n], dtype=torch.int32, device=dev), torch.tensor([n], dtype=torch.int32, device=dev)
    for window in (1, 40, 130):
        outs = [tdist.gqa_fwd_window_prefill(q, k, v, starts, lens, table, window=window) for _ in range(20)]
        check_status()
        for out in outs[1:]:
            assert torch.equal(out, outs[0])
        last = 300
        r, s = _exact(q[-last:], _keys(k, table[0], n), _keys(v, table[0], n), _mask(last, n, window, 0, dev), D ** -0.5, 0.0)
        _compare(outs[0][-last:], r, s, 2.0 ** -8)


@pytest.mark.parametrize("window,sinks", [(5, 2 ** 31), (5, 2 ** 32 + 1), (2 ** 32 + 1, 0)])
def test_settings_beyond_32_bits(cuda_device, window, sinks):
    """More first tokens, or a wider window, than any sequence is long: every key up to the query's position."""
    _prefill_case(cuda_device, "bf16", 8, 2, 128, 16, [(9, 50), (30, 200)], window, sinks)
    torch.manual_seed(1)
    k, v = _cache(20, 16, 2, 64, torch.bfloat16, cuda_device)
    q = torch.randn(2, 8, 64, device=cuda_device).to(torch.bfloat16)
    table, lens = torch.arange(20, dtype=torch.int32, device=cuda_device).view(2, 10), torch.tensor([160, 33], dtype=torch.int32, device=cuda_device)
    out = tdist.gqa_fwd_window_decode(q, k, v, lens, table, window=window, sinks=sinks)
    assert torch.equal(out, tdist.gqa_fwd_window_decode(q, k, v, lens, table))
