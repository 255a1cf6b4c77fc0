"""Serving operators where they can go wrong: calls interleaved on one stream, lengths and pages beyond the tensors, NaN and infinities,
tokens of no sequence, large soft caps, tables without a column, too many heads."""
import math

import pytest
import torch

import triton_distributed_b200 as tdist
from triton_distributed_b200.ops import flash_decode as FD
from triton_distributed_b200.ops import paged_attention as PA
from triton_distributed_b200.runtime import LocalWorld, check_status

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": (torch.bfloat16, 2.0 ** -8), "fp16": (torch.float16, 2.0 ** -11)}


def _pool(pages, page, Hkv, D, dt, dev):
    return torch.randn(pages, page, Hkv, D, device=dev).to(dt), torch.randn(pages, page, Hkv, D, device=dev).to(dt)


def _ints(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _exact(q, k, v, scale, cap=0.0, seen=None):
    """float64: q [n, Hq, D], k, v [keys, Hkv, D], seen [n, keys] (None: all) -> out, sum p |v|. NaN where the formula gives it."""
    n, Hq, D = q.shape
    Hkv = k.shape[1]
    s = torch.einsum("nhgd,khd->hgnk", q.double().view(n, Hkv, Hq // Hkv, D), k.double()) * scale
    if cap > 0:
        s = cap * torch.tanh(s / cap)
    if seen is not None:
        s = s.masked_fill(~seen, float("-inf"))
    p = torch.softmax(s, -1)
    both = [torch.einsum("hgnk,khd->nhgd", p, x).reshape(n, Hq, D) for x in (v.double(), v.double().abs())]
    return both[0], both[1]


def _keys(cache, table, n):
    return cache[table.long()].flatten(0, 1)[:n]


def _compare(out, ref, spread, u):
    """Within the bounds of test_paged_attention_gpu.py, and NaN exactly where the formula is."""
    assert torch.equal(out.isnan(), ref.isnan())
    bound = u * (spread + ref.abs()) + 1e-4 * spread + 1e-6
    worst = ((out.double() - ref).abs() - bound).nan_to_num(0.0).max()
    assert worst <= 0, float(worst)


def test_interleaved_shared_prefix_calls_on_one_stream(cuda_device, monkeypatch):
    """Two threads that call on one stream may launch prefix A, prefix B, own keys A, own keys B. Both own keys' launches use the stream's
    scratch, so the second must not begin before the first is done with it."""
    dev, page = cuda_device, 16
    torch.manual_seed(5)
    k, v = _pool(1200, page, 1, 128, torch.bfloat16, dev)
    calls = []
    for _ in range(2):
        order = torch.randperm(1200, device=dev).to(torch.int32)
        calls.append((torch.randn(1, 8, 128, device=dev).to(torch.bfloat16), k, v, _ints([700], dev), order[:44], _ints([16000], dev), order[44:1044].view(1, 1000)))
    want = [tdist.gqa_fwd_shared_prefix_decode(*c) for c in calls]
    torch.cuda.synchronize()
    attention, decode, kept, waiting = PA._run_attention, PA._run_decode, [], []

    def keep(*args):
        kept.append(args)   # each call's partials live until its own keys' launch, as in a thread of its own
        return attention(*args)

    monkeypatch.setattr(PA, "_run_attention", keep)
    monkeypatch.setattr(PA, "_run_decode", waiting.append)
    got = []
    for _ in range(100):
        got.append([tdist.gqa_fwd_shared_prefix_decode(*c) for c in calls])
        assert waiting[0].partial == waiting[1].partial and waiting[0].splits > 8   # one scratch, in global memory
        for a in waiting:
            decode(a)
        waiting.clear()
    check_status()
    for pair in got:
        assert all(torch.equal(a, b) for a, b in zip(pair, want))


@pytest.mark.parametrize("D,page", [(64, 16), (64, 1), (128, 16), (256, 64)])
@pytest.mark.parametrize("splits", [-1, 1, 16])
def test_lengths_beyond_the_table_are_cut(cuda_device, D, page, splits):
    """As many keys as the table has room for, whatever the length says; lengths below zero are none."""
    dev = cuda_device
    torch.manual_seed(D + page)
    room = 320 // page
    k, v = _pool(3 * room, page, 2, D, torch.bfloat16, dev)
    table = torch.randperm(3 * room, device=dev).view(3, room).to(torch.int32)
    q = torch.randn(3, 8, D, device=dev).to(torch.bfloat16)
    for window, sinks in ((None, 0), (100, 3)):
        args = dict(window=window, sinks=sinks, kv_split=splits)
        got = tdist.gqa_fwd_window_decode(q, k, v, _ints([321, 2 ** 31 - 1, -5], dev), table, **args)
        want = tdist.gqa_fwd_window_decode(q, k, v, _ints([320, 320, 0], dev), table, **args)
        check_status()
        assert torch.equal(got, want) and not got[2].any()
    pre = torch.randperm(3 * room, device=dev)[:room].to(torch.int32)
    got = tdist.gqa_fwd_shared_prefix_decode(q, k, v, 77, pre, _ints([1000, 320, -1], dev), table)
    want = tdist.gqa_fwd_shared_prefix_decode(q, k, v, 77, pre, _ints([320, 320, 0], dev), table)
    check_status()
    assert torch.equal(got, want)


@pytest.mark.parametrize("D,page", [(64, 16), (64, 1), (128, 16), (256, 64), (128, 3)])
@pytest.mark.parametrize("bad", [-1, 10 ** 9])
def test_pages_that_the_cache_does_not_have_read_as_zeros(cuda_device, D, page, bad):
    dev = cuda_device
    torch.manual_seed(D + page)
    room = -(-320 // page)
    k, v = _pool(2 * room + 1, page, 2, D, torch.bfloat16, dev)
    k[-1], v[-1] = 0, 0
    order = torch.randperm(2 * room, device=dev).view(2, room).to(torch.int32)
    wrong, zeros = order.clone(), order.clone()
    for i in (0, room // 2, room - 1):
        wrong[0, i], zeros[0, i] = bad, 2 * room
    q = torch.randn(2, 8, D, device=dev).to(torch.bfloat16)
    lens = _ints([315, 320], dev)
    for window, sinks in ((None, 0), (200, 3)):
        for splits in (-1, 1, 16):
            a, b = (tdist.gqa_fwd_window_decode(q, k, v, lens, t, window=window, sinks=sinks, kv_split=splits) for t in (wrong, zeros))
            check_status()
            assert torch.equal(a, b)
        a, b = (tdist.gqa_fwd_window_prefill(q, k, v, _ints([0, 1, 2], dev), lens, t, window=window, sinks=sinks) for t in (wrong, zeros))
        check_status()
        assert torch.equal(a, b)


def _spoil(what, q, k, v, at):
    """One value of sequence 1 that is no number, or infinite (scores of both infinities, and -inf alone, which weighs nothing)."""
    page, row = at
    if what == "q":
        q[1, 2, 5] = float("nan")
    elif what == "k":
        k[page, row, 0, 3] = float("nan")
    elif what == "v":
        v[page, row, 0, 3] = float("nan")
    elif what == "k inf":
        k[page, row, 0, 3] = float("inf")


@pytest.mark.parametrize("what", ["q", "k", "v", "k inf"])
@pytest.mark.parametrize("splits", [-1, 1, 3, 16])
@pytest.mark.parametrize("D,dtype", [(64, "fp16"), (128, "bf16"), (256, "bf16")])
def test_what_is_no_number_shows(cuda_device, what, splits, D, dtype):
    """A NaN, or an infinite score, in what a query sees makes its result NaN as the formula says, never a result over the other keys."""
    dev, (dt, u), page, n = cuda_device, DTYPES[dtype], 16, 700
    torch.manual_seed(D + splits)
    k, v = _pool(3 * 44 + 20, page, 2, D, dt, dev)
    order = torch.randperm(3 * 44 + 20, device=dev).to(torch.int32)
    table, pre = order[:132].view(3, 44), order[132:]
    q = torch.randn(3, 8, D, device=dev).to(dt)
    _spoil(what, q, k, v, (int(table[1, 40]), 7))   # key 647
    lens, scale = _ints([n, n, n], dev), D ** -0.5
    refs = [_exact(q[b:b + 1], _keys(k, table[b], n), _keys(v, table[b], n), scale) for b in range(3)]
    ref, spread = (torch.cat(t) for t in zip(*refs))
    assert ref[1].isnan().any() and not ref[0].isnan().any()
    for out in (tdist.gqa_fwd_window_decode(q, k, v, lens, table, kv_split=splits),
                tdist.gqa_fwd_batch_decode(q, k, v, None, None, lens, table, scale, kv_split=splits)):
        check_status()
        _compare(out, ref, spread, u)
    part = tdist.gqa_fwd_batch_decode_intra_rank(q, k, v, None, None, lens, table, scale, kv_split=splits)
    assert torch.equal(part[..., :D].isnan(), ref.isnan()) and torch.equal(part[..., D].isnan(), ref.isnan().all(-1))
    merged = FD.inter_rank_combine(torch.stack([part, part]), dt)
    check_status()
    assert torch.equal(merged.isnan(), ref.isnan())
    refs = [_exact(q[b:b + 1], torch.cat([_keys(k, pre, 300), _keys(k, table[b], n)]), torch.cat([_keys(v, pre, 300), _keys(v, table[b], n)]), scale)
            for b in range(3)]
    out = tdist.gqa_fwd_shared_prefix_decode(q, k, v, 300, pre, lens, table)
    check_status()
    _compare(out, *(torch.cat(t) for t in zip(*refs)), u)


def test_what_is_no_number_shows_on_every_rank(cuda_device):
    """The exchange of a sequence-parallel decode takes it along."""
    dev, world, B, Hq, Hkv, D = cuda_device, 2, 2, 8, 2, 128
    torch.manual_seed(2)
    lw = LocalWorld(world, dev)
    ctxs = [FD.create_sp_decode_context(r, world, B, Hq, D, heap=lw.heap(r), device=dev) for r in range(world)]
    q = torch.randn(B, Hq, D, device=dev).to(torch.bfloat16)
    lens = torch.full((world, B), 100, dtype=torch.int32, device=dev)
    shards = [(*_pool(14, 16, Hkv, D, torch.bfloat16, dev), torch.arange(14, dtype=torch.int32, device=dev).view(2, 7)) for _ in range(world)]
    shards[1][0][9, 0, 0, 0] = float("nan")   # rank 1, sequence 1, kv head 0
    for r in range(world):
        FD.sp_gqa_fwd_batch_decode(ctxs[r], q, shards[r][0], shards[r][1], lens, shards[r][2], phase=1)
    outs = [FD.sp_gqa_fwd_batch_decode(ctxs[r], q, shards[r][0], shards[r][1], lens, shards[r][2], phase=2) for r in range(world)]
    check_status()
    for out in outs:
        assert out[1, :4].isnan().all() and not out[1, 4:].isnan().any() and not out[0].isnan().any()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("kv_split", [-1, 1, 4])
@pytest.mark.parametrize("T,starts", [(300, [40, 100, 100, 250]), (34, [0, 33]), (34, [1, 34]), (65, [0, 64]), (500, [0, 1]), (90, [45, 45]), (40, [0, 0, 40])])
def test_tokens_of_no_sequence_give_zeros(cuda_device, D, kv_split, T, starts):
    """q padded to a fixed number of tokens, as for a captured graph: before the first sequence's and behind the last one's."""
    dev = cuda_device
    torch.manual_seed(T + D)
    B = len(starts) - 1
    k, v = _pool(B * 30, 16, 2, D, torch.bfloat16, dev)
    table = torch.randperm(B * 30, device=dev).view(B, 30).to(torch.int32)
    lens = _ints([450 - 50 * b for b in range(B)], dev)
    q = torch.randn(T, 8, D, device=dev).to(torch.bfloat16)
    first, last = starts[0], starts[-1]
    for window in (None, 60):
        out = torch.full_like(q, float("nan"))
        tdist.gqa_fwd_window_prefill(q, k, v, _ints(starts, dev), lens, table, window=window, out=out, kv_split=kv_split)
        check_status()
        assert not out[:first].any() and not out[last:].any()
        if last > first:
            alone = tdist.gqa_fwd_window_prefill(q[first:last], k, v, _ints([s - first for s in starts], dev), lens, table, window=window, kv_split=kv_split if kv_split > 0 else 2)
            torch.testing.assert_close(out[first:last].float(), alone.float(), atol=2.0 ** -6, rtol=2.0 ** -6)


def test_tokens_without_any_sequence_give_zeros(cuda_device):
    dev = cuda_device
    k, v = _pool(4, 16, 2, 64, torch.bfloat16, dev)
    q = torch.randn(5, 8, 64, device=dev).to(torch.bfloat16)
    out = torch.full_like(q, float("nan"))
    tdist.gqa_fwd_window_prefill(q, k, v, _ints([0], dev), _ints([], dev), torch.zeros((0, 4), dtype=torch.int32, device=dev), out=out)
    assert not out.any()


@pytest.mark.parametrize("cap", [65.0, 300.0, 1e3, 1e5, 1e8, 1e30, 3e38])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_large_soft_caps_change_little(cuda_device, cap, D):
    """The cap's error goes with the score, not with the cap: the bound is that of a call without one."""
    dev, page, n = cuda_device, 16, 900
    torch.manual_seed(D)
    k, v = _pool(3 * 57, page, 2, D, torch.float16, dev)
    order = torch.randperm(3 * 57, device=dev).to(torch.int32)
    table, pre = order[:114].view(2, 57), order[114:]
    scale = 3.5 * D ** -0.5   # scores of some 3.5
    q = torch.randn(140, 8, D, device=dev).to(torch.float16)
    seen = torch.arange(n, device=dev).view(1, -1) <= torch.arange(n - 70, n, device=dev).view(-1, 1)
    for loud in (False, True):
        if loud:
            q[3] *= 8000.0    # one token whose scores reach caps of 1e3 and more, in the tiles of the others
        refs = [_exact(q[70 * b:70 * b + 70], _keys(k, table[b], n), _keys(v, table[b], n), scale, cap, seen) for b in range(2)]
        ref, spread = (torch.cat(t) for t in zip(*refs))
        quiet = torch.arange(140, device=dev) != 3
        for split in (-1, 1, 3):
            out = tdist.gqa_fwd_window_prefill(q, k, v, _ints([0, 70, 140], dev), _ints([n, n], dev), table, scale=scale, soft_cap=cap, kv_split=split)
            check_status()
            assert out.isfinite().all()
            _compare(out[quiet], ref[quiet], spread[quiet], 2.0 ** -11)
    q = torch.randn(2, 8, D, device=dev).to(torch.float16)
    for loud in (False, True):
        if loud:
            q[0, 1] *= 8000.0   # a head beside the others of its MMA
        refs = [_exact(q[b:b + 1], _keys(k, table[b], n), _keys(v, table[b], n), scale, cap) for b in range(2)]
        both = [_exact(q[b:b + 1], torch.cat([_keys(k, pre, 500), _keys(k, table[b], n)]), torch.cat([_keys(v, pre, 500), _keys(v, table[b], n)]), scale, cap)
                for b in range(2)]
        quiet = torch.ones(2, 8, dtype=torch.bool, device=dev)
        quiet[0, 1] = not loud
        for split in (-1, 1, 16):
            out = tdist.gqa_fwd_window_decode(q, k, v, _ints([n, n], dev), table, scale=scale, soft_cap=cap, kv_split=split)
            pfx = tdist.gqa_fwd_shared_prefix_decode(q, k, v, 500, pre, _ints([n, n], dev), table, scale=scale, soft_cap=cap, kv_split=split)
            check_status()
            for got, want in ((out, refs), (pfx, both)):
                ref, spread = (torch.cat(t) for t in zip(*want))
                assert got.isfinite().all()
                _compare(got[quiet], ref[quiet], spread[quiet], 2.0 ** -11)


@pytest.mark.parametrize("scale,cap", [(1e-5, 1e-6), (1e-5, 30.0), (1e-9, 1e-9), (30.0, 1e-3), (2e4, 50.0), (1e-12, 1e3), (0.0, 1e4)])
def test_soft_caps_and_scales_of_any_size(cuda_device, scale, cap):
    """Also where the polynomial's coefficients leave fp32's range; masked scores on both sides of the window stay out."""
    dev, page, n, D = cuda_device, 16, 500, 64
    torch.manual_seed(7)
    k, v = _pool(32, page, 2, D, torch.float16, dev)
    table = torch.randperm(32, device=dev).view(1, 32).to(torch.int32)
    q = torch.randn(150, 8, D, device=dev).to(torch.float16)
    pos, j = torch.arange(n - 150, n, device=dev).view(-1, 1), torch.arange(n, device=dev).view(1, -1)
    seen = (j <= pos) & ((j > pos - 100) | (j < 3))
    ref, spread = _exact(q, _keys(k, table[0], n), _keys(v, table[0], n), scale, cap, seen)
    out = tdist.gqa_fwd_window_prefill(q, k, v, _ints([0, 150], dev), _ints([n], dev), table, window=100, sinks=3, scale=scale, soft_cap=cap)
    dec = tdist.gqa_fwd_window_decode(q[149:], k, v, _ints([n], dev), table, window=100, sinks=3, scale=scale, soft_cap=cap)
    check_status()
    _compare(out, ref, spread, 2.0 ** -11)
    _compare(dec, ref[149:], spread[149:], 2.0 ** -11)


def test_tables_without_a_column(cuda_device):
    """No own keys yet: the prefix alone. No keys at all: zeros."""
    dev = cuda_device
    torch.manual_seed(1)
    k, v = _pool(20, 16, 2, 128, torch.bfloat16, dev)
    q = torch.randn(3, 8, 128, device=dev).to(torch.bfloat16)
    pre, none, lens = torch.randperm(20, device=dev).to(torch.int32), torch.zeros((3, 0), dtype=torch.int32, device=dev), _ints([0, 0, 0], dev)
    got = tdist.gqa_fwd_shared_prefix_decode(q, k, v, 300, pre, lens, none)
    want = tdist.gqa_fwd_shared_prefix_decode(q, k, v, 300, pre, lens, pre[:3].view(3, 1))
    check_status()
    ref, spread = _exact(q, _keys(k, pre, 300), _keys(v, pre, 300), 128 ** -0.5)
    _compare(got, ref, spread, 2.0 ** -8)
    torch.testing.assert_close(got.float(), want.float(), atol=2.0 ** -8, rtol=2.0 ** -8)
    for out in (tdist.gqa_fwd_shared_prefix_decode(q, k, v, 0, pre[:0], lens, none), tdist.gqa_fwd_window_decode(q, k, v, lens, none, window=9),
                tdist.gqa_fwd_window_prefill(q, k, v, _ints([0, 1, 2, 3], dev), lens, none)):
        check_status()
        assert out.shape == q.shape and not out.any()


def test_refusals_of_many_heads_per_kv_head(cuda_device):
    dev = cuda_device
    k, v = _pool(8, 16, 1, 128, torch.bfloat16, dev)
    table, lens = torch.zeros(2, 4, dtype=torch.int32, device=dev), _ints([1, 1], dev)
    q = torch.zeros(2, 129, 128, dtype=torch.bfloat16, device=dev)
    with pytest.raises(ValueError, match="128 query heads"):
        tdist.gqa_fwd_window_prefill(q, k, v, _ints([0, 1, 2], dev), lens, table)
    with pytest.raises(ValueError, match="16 query heads"):
        tdist.gqa_fwd_shared_prefix_decode(q, k, v, 5, table[0], lens, table)
    with pytest.raises(ValueError, match="16 query heads"):
        tdist.gqa_fwd_window_decode(q, k, v, lens, table)
    with pytest.raises(ValueError, match="multiple of the kv heads"):
        tdist.gqa_fwd_window_decode(q, k[:, :, :0], v[:, :, :0], lens, table)
    with pytest.raises(ValueError, match="multiple of the kv heads"):
        tdist.gqa_fwd_window_decode(q[:, :0], k, v, lens, table)
    assert tdist.gqa_fwd_window_prefill(q[:, :128], k, v, _ints([0, 1, 2], dev), lens, table).shape == (2, 128, 128)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("split", [1, 4])
def test_prefill_passes_on_what_is_no_number_and_what_weighs_nothing(cuda_device, D, split):
    """A NaN key shows in the rows that see it and leaves those of other sequences alone; scores that are all -inf are like no keys."""
    dev = cuda_device
    torch.manual_seed(D)
    k, v = _pool(60, 16, 2, D, torch.bfloat16, dev)
    table = torch.randperm(60, device=dev).view(3, 20).to(torch.int32)
    q = torch.randn(300, 8, D, device=dev).to(torch.bfloat16).abs() + 0.1
    k[int(table[1, 19]), 15, 0, 0] = float("nan")         # sequence 1, its last key, kv head 0
    k[table[2].long(), :, 1, 0] = float("-inf")           # sequence 2, kv head 1
    out = tdist.gqa_fwd_window_prefill(q, k, v, _ints([0, 100, 200, 300], dev), _ints([320, 320, 320], dev), table, kv_split=split)
    check_status()
    assert out[199, :4].isnan().all() and not out[:100].isnan().any() and not out[100:200, 4:].isnan().any()
    assert not out[200:, 4:].any() and out[200:, :4].isfinite().all() and out[200:, :4].any()
    dec = tdist.gqa_fwd_window_decode(q[199:300:50].contiguous(), k, v, _ints([320] * 3, dev), table, kv_split=split)
    check_status()
    assert dec[1, :4].isnan().all() and not dec[2, 4:].any() and not dec[0].isnan().any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_an_infinite_temperature_on_a_gpu(cuda_device, dtype):
    """All finite logits weigh alike, those of -inf or NaN nothing; the same tokens as the statement's."""
    from triton_distributed_b200.ops.sampling import ref_sample_tokens
    torch.manual_seed(3)
    x = torch.randn(9, 30001, device=cuda_device).to(dtype)
    x[:, ::2] = -math.inf
    x[:, 5::10] = math.nan
    u = torch.linspace(0, 0.999, 9, device=cuda_device)
    for k, p, m in ((0, 1.0, 0.0), (0, 0.5, 0.0), (700, 0.9, 0.0), (0, 0.3, 0.5)):
        got, want = tdist.sample_tokens(x, u, math.inf, k, p, m), ref_sample_tokens(x, u, math.inf, k, p, m)
        check_status()
        assert torch.equal(got.tokens, want.tokens) and x.gather(1, got.tokens.long().view(-1, 1)).isfinite().all()
        torch.testing.assert_close(got.logprobs, want.logprobs, atol=1e-5, rtol=1e-5)
