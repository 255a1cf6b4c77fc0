"""GEMM of 8-bit integers with a scale per token and per output channel (``csrc/kernels/gemm_int8_sm100.cu``).

* ``quantize_int8_rowwise(x[M,K]) -> (int8 [M,K], fp32 [M])``: ``a = max(max|x|, 2^-100)``, ``scale = a / 127``, ``code = rint(x (127 / a))``; for
  activations row by row of every call, for weights ``[N,K]`` once
* ``gemm_int8(a, sa, b, sb, out_dtype) -> [M,N]``: ``C[m, n] = sa[m] sb[n] sum_k a[m, k] b[n, k]``

The sums are exact: 32-bit integers, K below 131072. A row that holds a NaN or an infinity is quantised to zeros with a scale of NaN, so its
results are NaN. Next to the block-scaled fp8 product (:mod:`.gemm_fp8`): half the scales' work on the tensor cores' full rate, where
one scale per row is enough for the activations.

CUDA tensors run the kernels (few rows: ``gemm_int8_skinny_sm100.cu``), CPU tensors the statements. Both calls take part in captured graphs.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from .. import _lib
from ..runtime import default_timeout_ns, global_status
from ..utils.profile import nvtx_range
from .quantized_cache import LEAST, quotient

launch_count = 0
MAX_K = 131071   # 128 x 128 x K stays below 2^31
MAX_ROWS = (1 << 31) - 512   # of either operand: rows are counted in 32 bits, whole tiles of them
_OUT = {torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16}
_ROWS = {**_OUT, torch.float32: _lib.DT_F32}


def ref_quantize_int8_rowwise(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    x = x.float()
    most = x.abs().amax(1, keepdim=True) if x.shape[1] else x.new_zeros((x.shape[0], 1))
    good = most < float("inf")   # (false for NaN)
    most = torch.where(good, most, 1.0).clamp_min(LEAST)
    codes = torch.where(good, torch.round(x * quotient(127.0, most)), 0.0).to(torch.int8)
    return codes, torch.where(good, quotient(most, 127.0), float("nan")).view(-1)


def ref_gemm_int8(a, sa, b, sb, out_dtype=torch.bfloat16) -> torch.Tensor:
    """Sums in fp64, which holds them exactly; scales and the result as the kernel rounds them."""
    acc = a.double() @ b.double().t()
    return (acc.float() * sa.float().view(-1, 1) * sb.float()).to(out_dtype)


def _call(index, fn, *args):
    """The native call with device ``index`` as the current one."""
    if index == torch._C._cuda_getDevice():
        return fn(*args)
    with torch.cuda.device(index):
        return fn(*args)


# What the checks found, by shapes, layouts, types and devices (never by addresses or contents): of a call's operands the arguments that they settle
_PLANS: dict = {}


def _remember(key, plan):
    if len(_PLANS) >= 4096:
        _PLANS.clear()
    _PLANS[key] = plan
    return plan


@nvtx_range("tdist.quantize_int8_rowwise")
def quantize_int8_rowwise(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``x [M, K]`` (bf16, fp16 or fp32; rows any distance apart) to int8 and one fp32 scale per row; K a multiple of 16."""
    global launch_count
    index = x.get_device()
    key = (x.shape, x.stride(), x.dtype)
    plan = _PLANS.get(key) if index >= 0 else None
    if plan is None:
        if x.dim() != 2 or x.shape[1] % 16 or x.shape[1] < 16:
            raise ValueError(f"expected [M, K] with K a multiple of 16, got {tuple(x.shape)}")
        if x.shape[0] >= 1 << 31 or x.shape[1] >= 1 << 31:
            raise ValueError("rows and their values are counted in 31 bits")
        if x.dtype not in _ROWS:
            raise TypeError("rows must be bf16, fp16 or fp32")
        if x.device.type != "cuda":
            return ref_quantize_int8_rowwise(x)
        plan = _remember(key, (x.shape[0], x.shape[1], x.stride(0), _ROWS[x.dtype], x.stride(1) == 1 and (x.stride(0) * x.element_size()) % 16 == 0))
    M, K, row, dtype, loads = plan
    if not loads or x.data_ptr() % 16:
        x, row = x.clone(memory_format=torch.contiguous_format), K
    codes, scale = x.new_empty(M, K, dtype=torch.int8), x.new_empty(M, dtype=torch.float32)
    if M:
        code = _call(index, _lib.lib().tdist_quant_int8_rowwise, x.data_ptr(), row, codes.data_ptr(), scale.data_ptr(), M, K, dtype,
                     torch._C._cuda_getCurrentRawStream(index))
        if code:
            _lib.check(code, "tdist_quant_int8_rowwise")
        launch_count += 1
    return codes, scale


def _check(a, sa, b, sb, out_dtype, out):
    if a.dim() != 2 or b.dim() != 2 or a.shape[1] != b.shape[1] or a.shape[1] % 16 or a.shape[1] < 16:
        raise ValueError(f"expected a[M,K], b[N,K] with K a multiple of 16, got {tuple(a.shape)} and {tuple(b.shape)}")
    if a.shape[1] > MAX_K:
        raise ValueError(f"K must be at most {MAX_K // 16 * 16}: longer sums may leave 32 bits")
    if a.shape[0] > MAX_ROWS or b.shape[0] > MAX_ROWS:
        raise ValueError(f"M and N must be at most {MAX_ROWS}")
    if b.shape[0] % 8:
        raise ValueError("N must be a multiple of 8")
    if a.dtype != torch.int8 or b.dtype != torch.int8:
        raise TypeError("operands must be int8")
    if sa.shape != a.shape[:1] or sb.shape != b.shape[:1]:
        raise ValueError(f"scales must be [M] and [N], got {tuple(sa.shape)} and {tuple(sb.shape)}")
    if sa.dtype != torch.float32 or sb.dtype != torch.float32:
        raise TypeError("scales must be fp32")
    if any(t.device != a.device for t in (sa, b, sb)):
        raise ValueError("operands and scales must be on one device")
    if out_dtype not in _OUT:
        raise TypeError("the result is bf16 or fp16")
    if any(not t.is_contiguous() for t in (a, b, sa, sb)):
        raise ValueError("operands and scales must be contiguous")
    if out is not None and (out.shape != (a.shape[0], b.shape[0]) or out.dtype != out_dtype or out.device != a.device or not out.is_contiguous()):
        raise ValueError("out must be contiguous [M, N] of out_dtype on the operands' device")


@nvtx_range("tdist.gemm_int8")
def gemm_int8(a: torch.Tensor, sa: torch.Tensor, b: torch.Tensor, sb: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``a [M, K]``, ``b [N, K]`` int8, ``sa [M]``, ``sb [N]`` fp32 -> ``[M, N]`` bf16 or fp16. K a multiple of 16, N of 8; M and N at most 2^31 - 512."""
    global launch_count
    index = a.get_device()
    key = (a.shape, b.shape, sa.shape, sb.shape, a.dtype, b.dtype, sa.dtype, sb.dtype, index, b.get_device(), sa.get_device(), sb.get_device(),
           a.is_contiguous() and b.is_contiguous() and sa.is_contiguous() and sb.is_contiguous(), out_dtype,
           None if out is None else (out.shape, out.is_contiguous(), out.dtype, out.get_device()))
    plan = _PLANS.get(key) if index >= 0 else None
    if plan is None:
        _check(a, sa, b, sb, out_dtype, out)
        if index < 0:
            c = ref_gemm_int8(a, sa, b, sb, out_dtype)
            return c if out is None else out.copy_(c)
        plan = _lib.GemmInt8Args()
        plan.m, plan.n, plan.k, plan.dtype = a.shape[0], b.shape[0], a.shape[1], _OUT[out_dtype]
        _remember(key, plan)
    c = out if out is not None else a.new_empty(plan.m, plan.n, dtype=out_dtype)
    if c.numel() == 0:
        return c
    g = _lib.GemmInt8Args.from_buffer_copy(plan)
    g.a, g.b, g.sa, g.sb, g.c = a.data_ptr(), b.data_ptr(), sa.data_ptr(), sb.data_ptr(), c.data_ptr()
    st = global_status()
    g.status = st.device_ptr if st is not None else None
    g.timeout_ns = default_timeout_ns()
    g.stream = torch._C._cuda_getCurrentRawStream(index)
    code = _call(index, _lib.lib().tdist_gemm_int8, C.byref(g))
    if code:
        _lib.check(code, "tdist_gemm_int8")
    launch_count += 1
    return c
