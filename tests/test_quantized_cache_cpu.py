"""A KV cache in 8 and 4 bits on CPU tensors: the plain statements against loops in Python floats, what quantising may cost, the
dispatcher's registrations, the checks of arguments."""
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import triton_distributed_b200 as tdist
import triton_distributed_b200.torch_ops  # noqa: F401
from triton_distributed_b200.ops import quantized_cache as QC


def _values(codes, scales, bits):
    """One row, in Python floats."""
    if bits == 8:
        return [(int(c) - 128) * float(scales) for c in codes]
    flat = [n for c in codes for n in (int(c) & 15, int(c) >> 4)]
    return [float(scales[i // 64, 1]) + float(scales[i // 64, 0]) * n for i, n in enumerate(flat)]


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantising_is_off_by_half_a_step(bits, dtype):
    """8 bits: half of a / 127 and fp32's roundings (2^-22 of the value's size). 4 bits: half a step, which is at most (max - least) / 15
    rounded up to 8 bits (2^-7 more), with least at most 2^-7 of its size below the minimum."""
    x = (torch.randn(40, 128, generator=torch.Generator().manual_seed(0)) * torch.logspace(-3, 3, 40).view(-1, 1) + 5.0).to(dtype)
    x[7] = 0.0
    codes, scales = QC.ref_quantize_rows(x, bits)
    for r in range(40):
        got = torch.tensor(_values(codes[r], scales[r], bits), dtype=torch.float64)
        want = x[r].double()
        if bits == 8:
            half = want.abs().max() / 254
        else:
            y = want.view(2, 64)
            half = ((y.amax(1) - y.amin(1) + 2.0 ** -7 * y.amin(1).abs()) / 30 * (1 + 2.0 ** -7)).repeat_interleave(64)
        assert bool(((got - want).abs() <= half + 2.0 ** -22 * want.abs().max() + 2.0 ** -100).all()), r
    assert torch.equal(QC.ref_dequantize_rows(codes, scales, bits)[3].double(), torch.tensor(_values(codes[3], scales[3], bits), dtype=torch.float64).float().double())


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("window,sinks,cap", [(None, 0, 0.0), (3, 0, 0.0), (1, 2, 5.0), (4, 9, 0.0)])
def test_write_read_and_decode_statements(bits, window, sinks, cap):
    g = torch.Generator().manual_seed(1)
    page, Hkv, G, D, lens = 3, 2, 2, 64, [9, 0, 4]
    cache = tdist.create_quantized_kv_cache(9, page, Hkv, D, bits, "cpu")
    assert cache.bits == bits and cache.head_dim == D
    table = torch.tensor([[4, 0, 7], [3, 3, 3], [8, 2, 1]], dtype=torch.int32)
    k, v = (torch.randn(13, Hkv, D, generator=g).to(torch.bfloat16) for _ in range(2))
    where = [(b, j) for b, n in enumerate(lens) for j in range(n)]
    slots = torch.tensor([int(table[b, j // page]) * page + j % page for b, j in where])
    tdist.kv_cache_write(cache, k, v, slots)
    rk, rv = tdist.kv_cache_read(cache, torch.tensor([1, 10, 12, 17]), torch.tensor(lens), table, 20, torch.float16)
    rows = {w: (1 if w[0] == 0 else 12) + w[1] for w in where}
    for t, w in enumerate(where):
        for h in range(Hkv):
            for x, r, i in ((k, rk, 0), (v, rv, 1)):
                c, s = QC.ref_quantize_rows(x[t, h], bits)
                assert torch.equal(r[rows[w], h], torch.tensor(_values(c, s, bits)).to(torch.float16))
    left = [i for i in range(20) if i not in rows.values()]
    assert (rk[left] == 0).all() and (rv[left] == 0).all()
    q = torch.randn(3, Hkv * G, D, generator=g)
    out = tdist.gqa_fwd_quantized_decode(q, cache, torch.tensor(lens), table, window=window, sinks=sinks, scale=0.1, soft_cap=cap)
    for b, n in enumerate(lens):
        seen = [j for j in range(n) if window is None or j >= n - window or j < sinks]
        for h in range(Hkv * G):
            keys, vals = ([_values(cache[i][table[b, j // page], j % page, h // G], cache[2 + i][table[b, j // page], h // G, j % page], bits)
                           for j in seen] for i in range(2))
            s = [0.1 * sum(float(x) * y for x, y in zip(q[b, h], key)) for key in keys]
            s = [cap * math.tanh(x / cap) if cap > 0 else x for x in s]
            p = [math.exp(x - max(s)) for x in s]
            ref = [sum(w * val[d] for w, val in zip(p, vals)) / sum(p) if p else 0.0 for d in range(D)]
            # fp32 sums of 64 products and a few keys
            torch.testing.assert_close(out[b, h].double(), torch.tensor(ref, dtype=torch.float64), atol=1e-5, rtol=1e-5)


@pytest.mark.parametrize("bits", [8, 4])
def test_bad_rows_and_places(bits):
    """NaN and infinities make their row (or group) NaN and no other; slots that are no place leave everything as it was."""
    cache = tdist.create_quantized_kv_cache(2, 4, 1, 128, bits, "cpu")
    x = torch.ones(4, 1, 128, dtype=torch.float16)
    x[1, 0, 5], x[2, 0, 100], x[3, 0, 0] = math.nan, math.inf, -math.inf
    tdist.kv_cache_write(cache, x, x, torch.tensor([0, 1, 2, 3]))
    k, _ = tdist.kv_cache_read(cache, torch.tensor([0, 4]), torch.tensor([4]), torch.tensor([[0]]), 4)
    bad = k[:, 0].isnan()
    assert not bad[0].any() and bad[1, :64].all() and bad[2, 64:].all() and bad[3, :64].all()
    if bits == 4:
        assert not bad[1, 64:].any() and not bad[2, :64].any()
    before = [t.clone() for t in cache]
    tdist.kv_cache_write(cache, x, x, torch.tensor([-1, 8, 1 << 40, -(1 << 40)]))
    tdist.kv_cache_write(cache, x[:0], x[:0], torch.zeros(0, dtype=torch.int64))
    assert all(torch.equal(a.nan_to_num(9.0), b.nan_to_num(9.0)) for a, b in zip(before, cache))
    # pages that the cache does not have read as zeros, lengths end with the table
    k, _ = tdist.kv_cache_read(cache, torch.tensor([0, 20]), torch.tensor([99]), torch.tensor([[7, -1]]), 20)
    assert (k == 0).all()
    q = torch.ones(1, 2, 128)
    assert (tdist.gqa_fwd_quantized_decode(q, cache, torch.tensor([8]), torch.tensor([[5, 9]])) == 0).all()
    assert (tdist.gqa_fwd_quantized_decode(q, cache, torch.tensor([0]), torch.tensor([[0, 1]])) == 0).all()
    assert (tdist.gqa_fwd_quantized_decode(q, cache, torch.tensor([5]), torch.zeros((1, 0), dtype=torch.int32)) == 0).all()


def test_dispatcher():
    for bits in (8, 4):
        cache = tdist.create_quantized_kv_cache(3, 4, 2, 64, bits, "cpu")
        k = torch.randn(5, 2, 64).to(torch.bfloat16)
        torch.ops.tdist.kv_cache_write(*cache, k, k, torch.arange(5))
        starts, lens, table = torch.tensor([0, 5]), torch.tensor([5]), torch.tensor([[0, 1]])
        a, b = torch.ops.tdist.kv_cache_read(*cache, starts, lens, table, 5, torch.bfloat16)
        want = tdist.kv_cache_read(cache, starts, lens, table, 5)
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])
        q = torch.randn(1, 4, 64)
        o = torch.ops.tdist.gqa_fwd_quantized_decode(q, *cache, lens, table, None, 0, 0.1, 0.0)
        assert torch.equal(o, tdist.gqa_fwd_quantized_decode(q, cache, lens, table, scale=0.1))
        with FakeTensorMode():
            fake = [torch.empty(t.shape, dtype=t.dtype) for t in cache]
            fs, fl, ft = torch.empty(2, dtype=torch.int32), torch.empty(1, dtype=torch.int32), torch.empty(1, 2, dtype=torch.int32)
            a, b = torch.ops.tdist.kv_cache_read(*fake, fs, fl, ft, 7, torch.float16)
            assert a.shape == (7, 2, 64) and b.dtype == torch.float16
            assert torch.ops.tdist.gqa_fwd_quantized_decode(torch.empty(1, 4, 64), *fake, fl, ft, None, 0, 0.1, 0.0).shape == (1, 4, 64)


def test_refusals():
    for bits in (16, 2):
        with pytest.raises(ValueError, match="8 or 4 bits"):
            tdist.create_quantized_kv_cache(2, 4, 2, 64, bits, "cpu")
    with pytest.raises(ValueError, match="multiple of 64"):
        tdist.create_quantized_kv_cache(2, 4, 2, 80, 8, "cpu")
    c8, c4 = (tdist.create_quantized_kv_cache(2, 4, 2, 64, bits, "cpu") for bits in (8, 4))
    k, slots = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.arange(3)
    lens, table, starts, q = torch.tensor([3]), torch.tensor([[0, 1]]), torch.tensor([0, 3]), torch.zeros(1, 4, 64)

    def write(cache=c8, k=k, v=k, slots=slots):
        tdist.kv_cache_write(cache, k, v, slots)

    def read(cache=c8, starts=starts, lens=lens, table=table, rows=3, dtype=torch.bfloat16, out=None):
        tdist.kv_cache_read(cache, starts, lens, table, rows, dtype, out)

    def decode(q=q, cache=c8, lens=lens, table=table, **kw):
        tdist.gqa_fwd_quantized_decode(q, cache, lens, table, **kw)

    for call in (write, read, decode):
        call()
        for bad, error in ((c8._replace(v=c8.v[:1]), ValueError), (c8._replace(k_scales=c8.k_scales[:, :1]), ValueError),
                           (c8._replace(k_scales=c4.k_scales), ValueError), (c4._replace(v_scales=c8.v_scales), ValueError),
                           (c8._replace(k=c8.k.to(torch.int8), v=c8.v.to(torch.int8)), TypeError), (c8._replace(k_scales=c8.k_scales.half()), TypeError),
                           (c8._replace(k=c8.k[0]), ValueError), (c8._replace(v=torch.empty(c8.v.shape, dtype=torch.uint8, device="meta")), ValueError)):
            with pytest.raises(error):
                call(cache=bad)
    for kw, error in (({"k": k[:2]}, ValueError), ({"v": k[:, :1]}, ValueError), ({"k": k.float(), "v": k.float()}, TypeError), ({"v": k.half()}, TypeError),
                      ({"slots": slots.float()}, TypeError), ({"slots": slots.view(1, 3)}, ValueError), ({"k": k.to("meta")}, ValueError)):
        with pytest.raises(error):
            write(**kw)
    good = torch.empty(3, 2, 64, dtype=torch.bfloat16)
    for kw, error in (({"starts": starts[:1]}, ValueError), ({"lens": lens.float()}, TypeError), ({"rows": -1}, ValueError), ({"rows": 1 << 31}, ValueError),
                      ({"dtype": torch.float32}, TypeError), ({"table": table[0]}, ValueError), ({"out": (good, good[:2])}, ValueError),
                      ({"out": (good, good.half())}, ValueError), ({"out": (good, good.transpose(0, 1))}, ValueError), ({"out": (good,)}, ValueError)):
        with pytest.raises(error):
            read(**kw)
    for kw, error in (({"q": q[..., :32]}, ValueError), ({"q": q[:, :3]}, ValueError), ({"window": 0}, ValueError), ({"sinks": -1}, ValueError),
                      ({"soft_cap": -1.0}, ValueError), ({"soft_cap": math.nan}, ValueError), ({"lens": torch.tensor([3, 3])}, ValueError),
                      ({"table": table.float()}, TypeError), ({"out": q[:, :2]}, ValueError), ({"q": q.to("meta")}, ValueError)):
        with pytest.raises(error):
            decode(**kw)


@pytest.mark.parametrize("wide", [False, True])
def test_the_ways_a_decode_is_dealt_out_are_ones_the_kernel_has(wide):
    """CTAs per sequence and head from 1 to 8, shares of at most 511 sequences that the machine has room for, or a small CTA each."""
    slots = 148 if wide else 296
    for B in (1, 2, 7, 64, 511, 512, 5000):
        for per_b in (1, 3, 8, 64, 500):
            for most in (0, 1, 17, 256, 1000, 6144, 6145, 524288, 1 << 30):
                for asked in (-1, 0, 1, 8, 9, 1000):
                    splits, shares = QC._decode_parts(B, per_b, most, max(most, 16), asked, slots, wide)
                    assert 0 <= splits <= 8 and shares >= 0 and not (splits and shares)
                    if shares:
                        assert B <= QC.MOST_SHARED and (shares == 1 or shares * per_b <= slots)
                    if 0 < asked <= 8:
                        assert splits == asked
