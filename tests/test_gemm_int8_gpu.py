"""GEMM of 8-bit integers: the sums are exact, and the three roundings behind them are IEEE's, so every result equals the statement
(sums in fp64, which holds whole numbers to 2^53) bit for bit; against 64 bits throughout, a bound."""
import math

import pytest
import torch

import triton_distributed_b200 as tdist
from triton_distributed_b200.ops import gemm_int8 as G8
from triton_distributed_b200.runtime import check_status

pytestmark = pytest.mark.gpu


def _operands(m, n, k, seed=0, full=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda r: torch.randint(-128, 128, (r, k), generator=g, device="cuda", dtype=torch.int8)   # noqa: E731
    a, b = new(m), new(n)
    if full:
        a.fill_(-128)
        b.fill_(-128)
    sa, sb = (torch.rand(r, generator=g, device="cuda") * 0.01 + 1e-4 for r in (m, n))
    return a, sa, b, sb


def _check(a, sa, b, sb, dtype):
    got = tdist.gemm_int8(a, sa, b, sb, out_dtype=dtype)
    check_status()
    want = G8.ref_gemm_int8(a, sa, b, sb, dtype)
    assert got.dtype == dtype and torch.equal(got, want), (got.float() - want.float()).abs().max()
    # one rounding of the sum, two of products, one of the result
    exact = (a.double() @ b.double().t()) * sa.double().view(-1, 1) * sb.double()
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    assert bool(((got.double() - exact).abs() <= exact.abs() * (half + 2.0 ** -22) + (2.0 ** -25 if dtype == torch.float16 else 0)).all())
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(1, 8, 16), (1, 4096, 4096), (3, 136, 48), (16, 6144, 1024), (17, 1000, 2064), (64, 512, 16384), (128, 4096, 512),
                                   (129, 264, 4096), (200, 4096, 144), (256, 256, 128), (257, 520, 272), (300, 1544, 4112), (1000, 5504, 4096),
                                   (1024, 2048, 8192), (2049, 776, 640), (511, 8, 1040), (4096, 4104, 528)])
def test_results_are_the_statement_bit_for_bit(m, n, k, dtype):
    _check(*_operands(m, n, k, seed=m + n), dtype)


@pytest.mark.parametrize("m,n,k", [(513, 3080, 2064), (2049, 4104, 528), (513, 7176, 1040), (2600, 7176, 4112), (2049, 4104, 4112), (1500, 5512, 144),
                                   (6200, 5512, 144), (6200, 12296, 144)])
def test_every_tiling(m, n, k):
    """Narrow and wide tiles of 256, 192 and 128 columns: one round and more of them, a last one in halves, odd last tiles."""
    _check(*_operands(m, n, k, seed=n), torch.bfloat16)


@pytest.mark.parametrize("m", [5, 300])
def test_the_longest_and_largest_sums(m):
    """-128 x -128 throughout at the largest K: 2147221504, 262144 below 2^31; cancelling sums beside them."""
    a, sa, b, sb = _operands(m, 264, G8.MAX_K // 16 * 16, full=True)
    b[::2] = 127
    b[5, ::2] = 127
    sa.fill_(2.0 ** -20)
    got = _check(a, sa, b, sb, torch.float16)
    assert (got[:, 1] > 0).all() and (got[:, 0] < 0).all()


@pytest.mark.parametrize("rows,k,dtype", [(1, 16, torch.bfloat16), (33, 4096, torch.bfloat16), (5, 16384, torch.float16), (7, 16400, torch.float32), (3, 65536, torch.bfloat16), (4097, 272, torch.float16)])
def test_quantised_rows_are_the_statement_bit_for_bit(rows, k, dtype):
    g = torch.Generator().manual_seed(k)
    x = (torch.randn(rows, k, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))).to(dtype)
    x[0, 0], x[rows // 2, k - 1] = 50.0, -77.0
    codes, scale = tdist.quantize_int8_rowwise(x.cuda())
    want = G8.ref_quantize_int8_rowwise(x)
    assert torch.equal(codes.cpu(), want[0]) and torch.equal(scale.cpu(), want[1])
    wide = torch.zeros(rows, k + 48, dtype=dtype)
    for at in (16, 5):      # a view with rows apart, on 16 bytes and off them
        wide[:, at:at + k] = x
        codes, scale = tdist.quantize_int8_rowwise(wide.cuda()[:, at:at + k])
        assert torch.equal(codes.cpu(), want[0]) and torch.equal(scale.cpu(), want[1])


def test_extreme_rows():
    x = torch.randn(8, 64, generator=torch.Generator().manual_seed(1))
    x[1] = 0.0
    x[2] *= 1e-37
    x[3] *= 1e37
    x[4, 9], x[5, 0], x[6, 63] = math.nan, math.inf, -math.inf
    x[7] = 2.0 ** -140
    want = G8.ref_quantize_int8_rowwise(x)
    codes, scale = tdist.quantize_int8_rowwise(x.cuda())
    assert torch.equal(codes.cpu(), want[0]) and torch.equal(scale.cpu().nan_to_num(-1.0), want[1].nan_to_num(-1.0))
    assert torch.equal(scale.isnan().cpu(), torch.tensor([False, False, False, False, True, True, True, False]))
    w, sw = tdist.quantize_int8_rowwise(torch.randn(16, 64, device="cuda"))
    y = tdist.gemm_int8(codes, scale, w, sw)
    assert y[4:7].isnan().all() and not y[:4].isnan().any() and (y[1] == 0).all()


def test_a_layer_in_a_captured_graph():
    """Quantise, multiply, again with the results; replayed on new rows."""
    g = torch.Generator(device="cuda").manual_seed(3)
    w1, s1 = tdist.quantize_int8_rowwise(torch.randn(1024, 512, generator=g, device="cuda"))
    w2, s2 = tdist.quantize_int8_rowwise(torch.randn(512, 1024, generator=g, device="cuda"))
    for m in (4, 300):
        x = torch.randn(m, 512, generator=g, device="cuda").to(torch.bfloat16)

        def layer():
            h = tdist.gemm_int8(*tdist.quantize_int8_rowwise(x), w1, s1)
            return tdist.gemm_int8(*tdist.quantize_int8_rowwise(h), w2, s2, out_dtype=torch.float16)

        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            layer()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer()
        for _ in range(3):
            x.normal_(generator=g)
            graph.replay()
            h = G8.ref_gemm_int8(*G8.ref_quantize_int8_rowwise(x.cpu()), w1.cpu(), s1.cpu())
            want = G8.ref_gemm_int8(*G8.ref_quantize_int8_rowwise(h), w2.cpu(), s2.cpu(), torch.float16)
            torch.cuda.synchronize()
            assert torch.equal(y.cpu(), want)
    check_status()


def test_two_streams_and_given_outputs():
    a, sa, b, sb = _operands(24, 2048, 4096)
    want = {m: G8.ref_gemm_int8(a[:m], sa[:m], b, sb) for m in (1, 24)}
    outs = [torch.full((m, 2048), 9.0, dtype=torch.bfloat16, device="cuda") for m in (1, 24) for _ in range(10)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i, o in enumerate(outs):
        with torch.cuda.stream(streams[i % 2]):
            m = o.shape[0]
            assert tdist.gemm_int8(a[:m], sa[:m], b, sb, out=o).data_ptr() == o.data_ptr()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[o.shape[0]]) for o in outs)
    check_status()
