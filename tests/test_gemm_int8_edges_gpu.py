"""Products of 8-bit integers at the ends of the scales' range, bit for bit against the statement (on the CPU, whose fp32 keeps subnormal numbers)."""
import pytest
import torch

import triton_distributed_b200 as tdist
from triton_distributed_b200.ops import gemm_int8 as G8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(3, 64, 256), (300, 512, 256), (2049, 4104, 144)])
def test_small_and_large_scales(m, n, k, dtype):
    """Results, and products of a sum with its first scale, that are subnormal in fp32; results beyond the type's range."""
    g = torch.Generator().manual_seed(m)
    a, b = (torch.randint(-128, 128, (r, k), generator=g, dtype=torch.int8) for r in (m, n))
    sa, sb = torch.exp2(torch.randint(-148, 100, (m,), generator=g).float()), torch.exp2(torch.randint(-60, 28, (n,), generator=g).float())
    sa[0], sb[:8] = 2.0 ** -120, torch.exp2(torch.arange(8).float() * -3)
    want = G8.ref_gemm_int8(a, sa, b, sb, dtype)
    assert bool(((want.float().abs() < 2.0 ** -126) & (want != 0)).any()) or dtype == torch.float16
    got = tdist.gemm_int8(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), out_dtype=dtype).cpu()
    assert torch.equal(got, want)
