"""The next token of every row of logits: temperature, top-k, top-p and min-p, at given random numbers.

``sample_tokens(logits[B,V], u[B], temperature, top_k, top_p, min_p) -> SampledTokens(tokens, logprobs, log_norm)``

A token's weight is ``round(2^31 exp((logit - max) / temperature))``, a whole number, so that every sum is exact and a draw does
not depend on how the row was split among the machine's processors. In the order of the logits, largest first and ties by index, the
filters keep: ``top_k`` the first k; ``top_p`` those before which less than p of the weight of these lies (always the first); ``min_p``
those of at least min_p of the largest weight. The token is the first one, in the order of the indices, at which the sum of
the kept weights passes ``floor(u x their sum)``.

CUDA tensors run ``csrc/kernels/sampling.cu`` (one launch), CPU tensors ``ref_sample_tokens``, the same in torch.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Union

import torch

from .. import _lib
from ..runtime import stream_ptr
from ..utils.profile import nvtx_range

launch_count = 0
ONE = 2147483648.0   # weight of a row's largest logit
_DTYPES = {torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16, torch.float32: _lib.DT_F32}
Setting = Union[float, int, torch.Tensor]


class SampledTokens(NamedTuple):
    tokens: torch.Tensor     # int32 [B], -1 where a row has no logit above -inf
    logprobs: torch.Tensor   # fp32 [B]: log of the token's share of the kept weights
    log_norm: torch.Tensor   # fp32 [B]: log of the sum of exp(logit / temperature) over the kept tokens (temperature 0: the largest logit)


def ref_sample_tokens(logits, u, temperature: Setting = 1.0, top_k: Setting = 0, top_p: Setting = 1.0, min_p: Setting = 0.0) -> SampledTokens:
    """The definition in torch operations: a full stable sort, cumulative sums of whole numbers."""
    B, V = logits.shape
    dev = logits.device

    def per_row(v, dtype):
        return (v if isinstance(v, torch.Tensor) else torch.full((B,), v, device=dev)).to(dtype).view(B, 1)

    t, k, p, m = per_row(temperature, torch.float32), per_row(top_k, torch.int64), per_row(top_p, torch.float32), per_row(min_p, torch.float32)
    x = logits.float()
    x = torch.where(torch.isnan(x), float("-inf"), x) + 0.0
    greedy = ~(t > 0)
    inv = 1.0 / torch.where(greedy, 1.0, t)
    top = x.amax(1, keepdim=True)
    below = x - top
    y = torch.where(x == top, 0.0, torch.where(below == float("-inf"), below, below * inv))   # (at an infinite temperature -inf x 0 is NaN)
    w = torch.round(torch.exp(y) * ONE).long()
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    keep = torch.arange(V, device=dev).view(1, -1) < torch.where(greedy, 1, torch.where(k <= 0, V, k))
    limit = torch.ceil(p.double() * (ws * keep).sum(1, keepdim=True).double()).clamp_min(1.0).long()
    keep &= (torch.cumsum(ws, 1) - ws < limit) | ~(p < 1)
    keep &= ws >= torch.ceil(m.double().clamp(0.0, 1.0) * ONE).long()
    kept = torch.zeros_like(w).scatter_(1, order, ws * keep)
    mass = kept.sum(1, keepdim=True)
    target = torch.minimum(torch.floor(u.double().view(B, 1) * mass.double()).long(), mass - 1)
    tokens = (torch.cumsum(kept, 1) > target).to(torch.int8).argmax(1, keepdim=True)
    norm = torch.log(mass.float() / ONE)
    none = top == float("-inf")
    return SampledTokens(torch.where(none, -1, tokens).view(B).to(torch.int32),
                         torch.where(none, float("-inf"), y.gather(1, tokens) - norm).view(B),
                         torch.where(none, float("-inf"), top * inv + norm).view(B))


_CHECKED: set = set()


def _check(logits, u, settings):
    if logits.dim() != 2 or u.shape != logits.shape[:1]:
        raise ValueError("logits must be [B, V] and u [B]")
    if logits.shape[1] < 1:
        raise ValueError("sampling needs at least one logit per row")
    if u.dtype != torch.float32 or logits.dtype not in _DTYPES:
        raise TypeError("u must be fp32, logits bf16, fp16 or fp32")
    if u.device != logits.device:
        raise ValueError("u must be on the logits' device")
    for name, v in zip(("temperature", "top_k", "top_p", "min_p"), settings):
        if isinstance(v, torch.Tensor):
            if v.shape != logits.shape[:1] or v.device != logits.device:
                raise ValueError(f"{name} must be a number or a tensor [B] on the logits' device")
            dtypes = (torch.int32, torch.int64) if name == "top_k" else (torch.float32,)
            if v.dtype not in dtypes:
                raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}")


@nvtx_range("tdist.sample_tokens")
def sample_tokens(logits: torch.Tensor, u: torch.Tensor, temperature: Setting = 1.0, top_k: Setting = 0, top_p: Setting = 1.0,
                  min_p: Setting = 0.0) -> SampledTokens:
    """``logits [B, V]`` (bf16, fp16 or fp32, any distance between rows), ``u`` fp32 ``[B]`` in [0, 1). Each setting is a number for
    all rows or a tensor ``[B]`` (fp32; ``top_k`` int32 or int64). Off: ``top_k <= 0``, ``top_p >= 1``, ``min_p <= 0``; ``temperature <= 0``
    (or NaN) takes the largest logit, the lowest index of equal ones. Logits of -inf or NaN are never drawn."""
    global launch_count
    given = (temperature, top_k, top_p, min_p)
    # the checks' outcome depends on shapes, types and devices only, and is kept by them
    key = (logits.shape, logits.dtype, logits.get_device(), u.shape, u.dtype, u.get_device(),
           tuple([(v.shape, v.dtype, v.get_device()) if isinstance(v, torch.Tensor) else None for v in given]))
    if key not in _CHECKED:
        _check(logits, u, given)
        if len(_CHECKED) >= 1024:
            _CHECKED.clear()
        _CHECKED.add(key)
    if logits.device.type != "cuda":
        return ref_sample_tokens(logits, u, temperature, top_k, top_p, min_p)
    B, V = logits.shape
    if logits.stride(1) != 1:
        logits = logits.contiguous()
    # one allocation, the tokens' bits among the floats
    tokens, logprobs, log_norm = torch.empty((3, B), dtype=torch.float32, device=logits.device).unbind()
    out = SampledTokens(tokens.view(torch.int32), logprobs, log_norm)
    if B == 0:
        return out
    a = _lib.SampleArgs()
    a.logits, a.stride, a.B, a.V, a.dtype = logits.data_ptr(), logits.stride(0), B, V, _DTYPES[logits.dtype]
    if not u.is_contiguous():
        u = u.contiguous()
    a.u = u.data_ptr()
    # tensors are read by the row, numbers serve all rows; copies outlive the launch call in these names
    if isinstance(temperature, torch.Tensor):
        temperature = temperature.contiguous()
        a.temperature = temperature.data_ptr()
    else:
        a.one_temperature = temperature
    if isinstance(top_k, torch.Tensor):
        top_k = (top_k if top_k.dtype == torch.int32 else top_k.clamp(0, V).to(torch.int32)).contiguous()
        a.top_k = top_k.data_ptr()
    else:
        a.one_top_k = max(0, min(int(top_k), V))
    if isinstance(top_p, torch.Tensor):
        top_p = top_p.contiguous()
        a.top_p = top_p.data_ptr()
    else:
        a.one_top_p = top_p
    if isinstance(min_p, torch.Tensor):
        min_p = min_p.contiguous()
        a.min_p = min_p.data_ptr()
    else:
        a.one_min_p = min_p
    a.tokens, a.logprobs, a.log_norm = out.tokens.data_ptr(), logprobs.data_ptr(), log_norm.data_ptr()
    a.stream = stream_ptr(logits.device)
    code = _lib.lib().tdist_sample(C.byref(a))
    if code:
        _lib.check(code, "tdist_sample")
    launch_count += 1
    return out
