"""GEMM of 8-bit integers without a GPU: the statements against loops in whole numbers, the schedule, the checks of arguments."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import triton_distributed_b200 as tdist
import triton_distributed_b200.torch_ops  # noqa: F401
from triton_distributed_b200 import _lib


def test_statements():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 32, generator=g).to(torch.bfloat16)
    codes, scale = tdist.quantize_int8_rowwise(x)
    for r in range(3):
        most = max(abs(float(v)) for v in x[r])
        assert float(scale[r]) == pytest.approx(most / 127, rel=2.0 ** -23)
        for c in range(32):   # half a step and the quotient's roundings
            assert abs(int(codes[r, c]) - float(x[r, c]) * 127 / most) <= 0.5 + 2.0 ** -15
    w, sw = torch.randint(-128, 128, (8, 32), generator=g, dtype=torch.int8), torch.rand(8, generator=g)
    y = tdist.gemm_int8(codes, scale, w, sw, out_dtype=torch.float16)
    for r in range(3):
        for n in range(8):
            acc = sum(int(p) * int(q) for p, q in zip(codes[r], w[n]))
            assert float(y[r, n]) == pytest.approx(acc * float(scale[r]) * float(sw[n]), rel=2.0 ** -11 + 2.0 ** -22, abs=2.0 ** -25)
    out = torch.empty(3, 8, dtype=torch.float16)
    assert tdist.gemm_int8(codes, scale, w, sw, out_dtype=torch.float16, out=out) is out and torch.equal(out, y)


@pytest.mark.parametrize("wide", [0, 1])
def test_every_tile_is_dealt_once(wide):
    check = _lib.lib().tdist_gemm_int8_schedule_check
    for units in (1, 2, 7, 73, 74):
        for m_tiles in (1, 2, 8, 9, 33):
            for n_tiles in (1, 2, 3, 21, 56):
                assert check(wide, units, m_tiles, n_tiles) == 0, (units, m_tiles, n_tiles)


def test_refusals():
    a, b = torch.zeros(4, 32, dtype=torch.int8), torch.zeros(8, 32, dtype=torch.int8)
    sa, sb = torch.ones(4), torch.ones(8)
    tdist.gemm_int8(a, sa, b, sb)
    long_a, long_b = torch.zeros(1, 131072, dtype=torch.int8), torch.zeros(8, 131072, dtype=torch.int8)
    for args, error in (((a[:, :24], sa, b[:, :24], sb), ValueError), ((a, sa, b[:, :16], sb), ValueError), ((a, sa, b[:7], sb[:7]), ValueError),
                        ((a.float(), sa, b, sb), TypeError), ((a, sa, b.to(torch.uint8), sb), TypeError), ((a, sa[:3], b, sb), ValueError),
                        ((a, sa, b, sb.view(8, 1)), ValueError), ((a, sa.half(), b, sb), TypeError), ((a, sa.to("meta"), b, sb), ValueError),
                        ((a.t().contiguous().t(), sa, b, sb), ValueError), ((a[0], sa, b, sb), ValueError), ((long_a, sa[:1], long_b, sb), ValueError)):
        with pytest.raises(error):
            tdist.gemm_int8(*args)
    for kw, error in (({"out_dtype": torch.float32}, TypeError), ({"out": torch.zeros(4, 8)}, ValueError), ({"out": torch.zeros(8, 4, dtype=torch.bfloat16).t()}, ValueError)):
        with pytest.raises(error):
            tdist.gemm_int8(a, sa, b, sb, **kw)
    for x, error in ((torch.zeros(4, 24), ValueError), (torch.zeros(32), ValueError), (torch.zeros(4, 0), ValueError), (torch.zeros(4, 32, dtype=torch.float64), TypeError)):
        with pytest.raises(error):
            tdist.quantize_int8_rowwise(x)


def test_dispatcher():
    x, w = torch.randn(5, 32), torch.randn(16, 32)
    a, sa = torch.ops.tdist.quantize_int8_rowwise(x)
    b, sb = torch.ops.tdist.quantize_int8_rowwise(w)
    assert torch.equal(torch.ops.tdist.gemm_int8(a, sa, b, sb, torch.float16), tdist.gemm_int8(a, sa, b, sb, out_dtype=torch.float16))
    with FakeTensorMode():
        a, sa = torch.ops.tdist.quantize_int8_rowwise(torch.empty(5, 32))
        assert a.dtype == torch.int8 and sa.shape == (5,)
        y = torch.ops.tdist.gemm_int8(a, sa, torch.empty(16, 32, dtype=torch.int8), torch.empty(16), torch.bfloat16)
        assert y.shape == (5, 16) and y.dtype == torch.bfloat16
