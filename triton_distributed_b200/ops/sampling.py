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
    greedy = t <= 0
    inv = 1.0 / torch.where(greedy, 1.0, t)
    top = x.amax(1, keepdim=True)
    y = torch.where(x == top, 0.0, (x - top) * inv)
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


@nvtx_range("tdist.sample_tokens")
def sample_tokens(logits: torch.Tensor, u: torch.Tensor, temperature: Setting = 1.0, top_k: Setting = 0, top_p: Setting = 1.0,
                  min_p: Setting = 0.0) -> SampledTokens:
    """``logits [B, V]`` (bf16, fp16 or fp32, any distance between rows), ``u`` fp32 ``[B]`` in [0, 1). Each setting is a number for
    all rows or a tensor ``[B]`` (fp32; ``top_k`` int32 or int64). Off: ``top_k <= 0``, ``top_p >= 1``, ``min_p <= 0``; ``temperature <= 0``
    takes the largest logit, the lowest index of equal ones. Logits of -inf or NaN are never drawn."""
    global launch_count
    if logits.dim() != 2 or u.shape != logits.shape[:1]:
        raise ValueError("logits must be [B, V] and u [B]")
    B, V = logits.shape
    if V < 1:
        raise ValueError("sampling needs at least one logit per row")
    if u.dtype != torch.float32 or logits.dtype not in _DTYPES:
        raise TypeError("u must be fp32, logits bf16, fp16 or fp32")
    for name, v, dtypes in (("temperature", temperature, (torch.float32,)), ("top_k", top_k, (torch.int32, torch.int64)),
                            ("top_p", top_p, (torch.float32,)), ("min_p", min_p, (torch.float32,))):
        if isinstance(v, torch.Tensor):
            if v.shape != (B,) or v.device != logits.device:
                raise ValueError(f"{name} must be a number or a tensor [B] on the logits' device")
            if v.dtype not in dtypes:
                raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}")
    if u.device != logits.device:
        raise ValueError("u must be on the logits' device")
    if logits.device.type != "cuda":
        return ref_sample_tokens(logits, u, temperature, top_k, top_p, min_p)
    if logits.stride(1) != 1:
        logits = logits.contiguous()
    out = SampledTokens(torch.empty(B, dtype=torch.int32, device=logits.device), torch.empty(B, dtype=torch.float32, device=logits.device),
                        torch.empty(B, dtype=torch.float32, device=logits.device))
    if B == 0:
        return out
    a = _lib.SampleArgs()
    held = []   # copies that have to outlive the launch call

    def per_row(v, dtype):
        if not isinstance(v, torch.Tensor):
            return None
        if dtype == torch.int32 and v.dtype == torch.int64:
            v = v.clamp(0, V)
        v = v.to(dtype).contiguous()
        held.append(v)
        return v.data_ptr()

    a.logits, a.u = logits.data_ptr(), per_row(u, torch.float32)
    a.temperature, a.top_k = per_row(temperature, torch.float32), per_row(top_k, torch.int32)
    a.top_p, a.min_p = per_row(top_p, torch.float32), per_row(min_p, torch.float32)
    a.one_temperature = 0.0 if a.temperature is not None else float(temperature)
    a.one_top_k = 0 if a.top_k is not None else max(0, min(int(top_k), V))
    a.one_top_p = 0.0 if a.top_p is not None else float(top_p)
    a.one_min_p = 0.0 if a.min_p is not None else float(min_p)
    a.tokens, a.logprobs, a.log_norm = out.tokens.data_ptr(), out.logprobs.data_ptr(), out.log_norm.data_ptr()
    a.stride, a.B, a.V, a.dtype = logits.stride(0), B, V, _DTYPES[logits.dtype]
    a.stream = stream_ptr(logits.device)
    _lib.check(_lib.lib().tdist_sample(C.byref(a)), "tdist_sample")
    launch_count += 1
    return out
