"""The quantised cache at the ends of its types' ranges, by the plain statements."""
import math

import pytest
import torch

import triton_distributed_b200 as tdist
from triton_distributed_b200.ops import quantized_cache as QC


def wide_rows():
    """Groups of bf16 whose range is beyond fp32's largest number, and groups just within."""
    x = torch.randn(8, 1, 64, generator=torch.Generator().manual_seed(1))
    x[0, 0, ::2], x[0, 0, 1::2] = 3.3e38, -3.3e38
    x[1] = x[1].clamp(-3, 3) / 3 * 3.38e38
    x[1, 0, 0], x[1, 0, 1] = -3.38e38, 3.38e38
    x[2], x[2, 0, 3], x[2, 0, 4] = 0.0, 3.38e38, -1e37
    x[3], x[3, 0, 3], x[3, 0, 4] = 1e-30, -3.38e38, 3e37
    x[4] = x[4].abs() * 2.0 ** 125 / 4
    x[5, 0, 9], x[5, 0, 10] = 1.7e38, -1.7e38
    x[6], x[6, 0, 1] = -torch.finfo(torch.bfloat16).max, torch.finfo(torch.bfloat16).max
    return x.to(torch.bfloat16)


def test_groups_whose_range_is_beyond_fp32():
    """4 bits: half a step, at most (max - least) / 30 and 2^-7 of it, and the codes' roundings, in 64 bits."""
    x = wide_rows()
    codes, pairs = QC.ref_quantize_rows(x, 4)
    assert bool(pairs.isfinite().all())
    step, least = pairs.double()[..., 0], pairs.double()[..., 1]
    y = x.double()
    assert bool((least <= y.amin(-1)[..., None]).all()) and bool((step * 15 >= (y.amax(-1)[..., None] - least) * (1 - 2.0 ** -22)).all())
    assert bool((step <= ((y.amax(-1)[..., None] - least) / 15) * (1 + 2.0 ** -7)).all())
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double()
    assert bool(((c * step + least - y).abs() <= step * (0.5 + 2.0 ** -18)).all())


def largest_rows(dtype):
    """Groups that reach the type's largest numbers, of either sign, and beyond (8: read in a narrower type)."""
    most = torch.finfo(dtype).max
    x = torch.randn(9, 1, 64, generator=torch.Generator().manual_seed(2)).clamp(-4, 4) / 4 * most
    x[0, 0, ::2], x[0, 0, 1::2] = most, 0.0
    x[1, 0, ::2], x[1, 0, 1::2] = -most, 0.0
    x[2], x[2, 0, 5], x[2, 0, 6] = most / 2, most, -most
    x[3] = -most
    x[4], x[4, 0, 7] = most * 0.997, -most * 0.998
    x[5] = x[5].abs()
    x[6] = -x[6].abs()
    x[7] = 1.0
    return x.to(dtype)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_finite_rows_read_as_finite(bits, dtype):
    """And no further off than half a step, which saturating only lessens; a type's rounding in 8 bits, where half a step is 2^-8 of the largest."""
    x = torch.cat([largest_rows(dtype), wide_rows()]) if dtype == torch.bfloat16 else largest_rows(dtype)
    n = x.shape[0]
    cache = tdist.create_quantized_kv_cache(1, n, 1, 64, bits, "cpu")
    tdist.kv_cache_write(cache, x, x, torch.arange(n))
    k, v = tdist.kv_cache_read(cache, torch.tensor([0, n]), torch.tensor([n]), torch.tensor([[0]]), n, dtype)
    assert torch.equal(k, v) and bool(k.isfinite().all())
    most = x.double().abs().amax(-1, keepdim=True)
    half = most / 254 if bits == 8 else cache.k_scales.double()[0, 0, :, :, 0].unsqueeze(1) / 2
    assert bool(((k.double() - x.double()).abs() <= half * (1 + 2.0 ** -16) + most * torch.finfo(dtype).eps / 2).all())


def test_what_does_not_fit_a_narrower_type_is_infinite():
    """Numbers of bf16 read as fp16: 10^6 lies beyond by more than half a step of its group, 65536 by less."""
    x = torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    x[0, 0, :2] = torch.tensor([1e6, -1e6])
    x[1] = 65536.0
    x[1, 0, 0] = 60000.0
    cache = tdist.create_quantized_kv_cache(1, 2, 1, 64, 4, "cpu")
    tdist.kv_cache_write(cache, x, x, torch.arange(2))
    k, _ = tdist.kv_cache_read(cache, torch.tensor([0, 2]), torch.tensor([2]), torch.tensor([[0]]), 2, torch.float16)
    assert k[0, 0, 0] == math.inf and k[0, 0, 1] == -math.inf and bool(k[0, 0, 2:].isfinite().all()) and bool(k[1].isfinite().all())


def test_sizes_beyond_32_bits_are_refused():
    """Views of one element; the native arguments are 32 bits wide and would be cut."""
    many = 1 << 32
    one = lambda dtype, *shape: torch.zeros((1,) * len(shape), dtype=dtype).expand(*shape)   # noqa: E731
    for shape in ((1, many + 16), (1, 1 << 31), (1 << 31, 16)):
        with pytest.raises(ValueError, match="31 bits"):
            tdist.quantize_int8_rowwise(one(torch.bfloat16, *shape))
    a, b, sa, sb = one(torch.int8, 4, 16), one(torch.int8, 8, 16), torch.ones(4), torch.ones(8)
    for m in (many + 4, (1 << 31) - 256):
        with pytest.raises(ValueError, match="at most"):
            tdist.gemm_int8(one(torch.int8, m, 16), one(torch.float32, m), b, sb)
        with pytest.raises(ValueError, match="at most"):
            tdist.gemm_int8(a, sa, one(torch.int8, m, 16), one(torch.float32, m))
    cache = tdist.create_quantized_kv_cache(2, 4, 1, 64, 8, "cpu")
    lens, wide = torch.tensor([3]), one(torch.int32, 1, many + 1)
    with pytest.raises(ValueError, match="31 bits"):
        tdist.gqa_fwd_quantized_decode(torch.zeros(1, 2, 64), cache, lens, wide)
    with pytest.raises(ValueError, match="31 bits"):
        tdist.kv_cache_read(cache, torch.tensor([0, 3]), lens, wide, 3)


def test_lengths_end_with_what_is_counted():
    cache = tdist.create_quantized_kv_cache(1, 1 << 20, 1, 64, 8, "cpu")
    table = torch.zeros((1, 1), dtype=torch.int32).expand(1, 1 << 11)
    assert QC._limits(cache, table, torch.tensor([(1 << 31) - 1])) == [(1 << 31) - 64] and QC._limits(cache, table, torch.tensor([77])) == [77]
    assert QC._limits(cache, table[:, :3], torch.tensor([1 << 40])) == [3 << 20]
