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
