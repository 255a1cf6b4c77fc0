"""Attention over the paged KV cache beyond plain decode: sliding windows with first tokens that stay visible (sinks), prefill of
a ragged batch, and decode of a batch whose sequences share a prefix.

* ``gqa_fwd_window_decode(q[B,Hq,D], k_cache[blocks,page,Hkv,D], v_cache, kv_lens[B], block_table[B,max_blocks], window, sinks,
  scale, soft_cap) -> [B,Hq,D]``: the query of a sequence of n keys sees key j if j >= n - window or j < sinks
* ``gqa_fwd_window_prefill(q[T,Hq,D], k_cache, v_cache, q_starts[B+1], kv_lens[B], block_table, window, sinks, scale,
  soft_cap) -> [T,Hq,D]``: tokens ``q_starts[b]:q_starts[b+1]`` are the last positions of sequence b, whose keys (theirs among
  them) are in the cache already; position p sees key j if j <= p and (j > p - window or j < sinks)
* ``gqa_fwd_shared_prefix_decode(q[B,Hq,D], k_cache, v_cache, prefix_len[1], prefix_table[max_blocks], kv_lens[B],
  block_table, scale, soft_cap) -> [B,Hq,D]``: the softmax runs over the keys of the prefix, read once for all, and the sequence's own

``window=None`` is no limit: plain causal attention. A query that sees no key (or none whose score is above -inf) gives zeros, and so does
a token that ``q_starts`` (which must not decrease) gives to no sequence, as in a batch padded for a captured graph. Pages without a
visible key are not read, nor are their table entries (a server may have given them back). What lies in a page behind a sequence's last
key may be anything; keys that only some of a sequence's queries see have to be finite, as 0 x NaN is NaN in every query's sum. A NaN that
a query sees makes its result NaN. On a GPU lengths are cut to what the table has room for, and a page that the cache does not have reads
as zeros: nothing outside the tensors is touched.

Decode runs the split decode kernel (``csrc/kernels/flash_decode.cu``), prefill and the shared prefix the tcgen05 kernel
(``csrc/kernels/attention_sm100.cu``). CPU tensors run ``ref_window_attn`` / ``ref_shared_prefix_attn``, the plain statements.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional

import torch

from .. import _lib
from ..runtime import default_timeout_ns, global_status, stream_ptr
from ..utils.profile import nvtx_range
from . import flash_decode as FD

launch_count = 0
_DTYPES = {torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16}
NO_WINDOW = 0x7FFFFFFF


def _attend(q, k, v, seen, scale, soft_cap):
    """fp32 attention of q [n, Hq, D] over k, v [keys, Hkv, D] with a mask [n, keys]; zeros where a row sees nothing above -inf."""
    n, Hq, D = q.shape
    Hkv = k.shape[1]
    s = torch.einsum("nhgd,khd->hgnk", q.float().view(n, Hkv, Hq // Hkv, D), k.float()) * scale
    if soft_cap > 0:
        s = soft_cap * torch.tanh(s / soft_cap)
    s = s.masked_fill(~seen, float("-inf"))
    p = torch.softmax(s, dim=-1).masked_fill((s == float("-inf")).all(-1, keepdim=True), 0.0)
    return torch.einsum("hgnk,khd->nhgd", p, v.float()).reshape(n, Hq, D)


def ref_window_attn(q, k_cache, v_cache, q_starts, kv_lens, block_table, window=None, sinks: int = 0, scale=None, soft_cap: float = 0.0):
    """fp32 reference, sequence by sequence: keys gathered from their pages, an explicit mask."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    page = k_cache.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float32, device=q.device)
    for b in range(kv_lens.shape[0]):
        q0, q1, kv = int(q_starts[b]), int(q_starts[b + 1]), int(kv_lens[b])
        if q1 <= q0 or kv <= 0:
            continue
        pos = torch.arange(kv - (q1 - q0), kv, device=q.device).unsqueeze(1)
        j = torch.arange(kv, device=q.device)
        seen = j <= pos
        if window is not None:
            seen = seen & ((j > pos - window) | (j < sinks))
        at = j[seen.any(0)]
        pages = block_table[b][at // page].long()
        out[q0:q1] = _attend(q[q0:q1], k_cache[pages, at % page], v_cache[pages, at % page], seen[:, at], scale, soft_cap)
    return out


def ref_shared_prefix_attn(q, k_cache, v_cache, prefix_len, prefix_table, kv_lens, block_table, scale=None, soft_cap: float = 0.0):
    """fp32 reference: every sequence's keys are the prefix' and its own, one after the other."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    page, P = k_cache.shape[1], int(prefix_len)
    at = torch.arange(P, device=q.device)
    pages, rows = prefix_table[at // page].long(), at % page
    out = torch.zeros(q.shape, dtype=torch.float32, device=q.device)
    for b in range(q.shape[0]):
        own = torch.arange(int(kv_lens[b]), device=q.device)
        pg, rw = torch.cat([pages, block_table[b][own // page].long()]), torch.cat([rows, own % page])
        if pg.numel():
            seen = torch.ones((1, pg.numel()), dtype=torch.bool, device=q.device)
            out[b:b + 1] = _attend(q[b:b + 1], k_cache[pg, rw], v_cache[pg, rw], seen, scale, soft_cap)
    return out


def _check(q, k_cache, v_cache, window, sinks, soft_cap, ints, most_heads):
    """``most_heads``: query heads per kv head that the operator's kernels take."""
    if q.dim() != 3 or k_cache.dim() != 4:
        raise ValueError("q must be [tokens, Hq, D], the caches [blocks, page, Hkv, D]")
    if k_cache.shape != v_cache.shape or k_cache.shape[3] != q.shape[2]:
        raise ValueError("k and v caches need the same shape, with head_dim == q's")
    if k_cache.shape[2] < 1 or q.shape[1] < 1 or q.shape[1] % k_cache.shape[2]:
        raise ValueError("the query heads must be a multiple of the kv heads")
    if window is not None and window < 1:
        raise ValueError("the window must be at least 1 (None: no limit)")
    if sinks < 0 or not soft_cap >= 0:
        raise ValueError("sinks and soft_cap must not be negative")
    for name, t, shape in ints:
        if t.dim() != len(shape) or any(s is not None and s != n for s, n in zip(shape, t.shape)):
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {['any' if s is None else s for s in shape]}")
        if t.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"{name} must hold integers (int32 or int64)")
        if t.device != q.device:
            raise ValueError(f"{name} must be on q's device")
    if k_cache.device != q.device or v_cache.device != q.device:
        raise ValueError("q and the caches must be on one device")
    if q.device.type != "cuda":
        return
    if q.dtype not in _DTYPES or k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        raise TypeError("q, k_cache and v_cache must share one of bf16 / fp16")
    if q.shape[1] > most_heads * k_cache.shape[2]:
        raise ValueError(f"at most {most_heads} query heads per kv head")
    if q.shape[2] not in (64, 128, 256):
        raise ValueError("head_dim must be 64, 128 or 256")
    if k_cache.stride(3) != 1 or v_cache.stride() != k_cache.stride() or q.stride(2) != 1:
        raise ValueError("q and the caches must have a contiguous head dimension, the caches equal strides")


def _output(out, q):
    if out is None:
        return torch.empty_like(q) if q.is_contiguous() else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or not out.is_contiguous():
        raise ValueError("out must be contiguous, of q's shape, dtype and device")
    return out


def _stated(ref, q, out):
    """What a plain statement gave, as the result of the call."""
    return ref.to(q.dtype) if out is None else _output(out, q).copy_(ref)


def _int32(t):
    return (t if t.dtype == torch.int32 else t.to(torch.int32)).contiguous()


def _splits(ctas: int, keys: int, head_dim: int, sms: int) -> int:
    """Parts that the keys of a row tile are cut into: as many CTAs as the machine has SMs (one fits an SM), but at least 256 keys
    (512 with head_dim 256) each: below that the parts' merge costs about what it saves (8 sequences, prefix of 2048, heads of 128, parts of 512 / 256 / 114
    keys 20.8 / 17.8 / 19.5 us; 201 sequences, 5003, heads of 256, parts of 834 / 500 / 357 keys 59.1 / 56.7 / 55.7 us)."""
    return max(1, min(sms // max(1, ctas), -(-keys // (256 if head_dim <= 128 else 512)), 200))


# What a call works out from its tensors' shapes, strides and types and its settings (never from their addresses or contents): checks,
# splits, and the native arguments but for the pointers. Bounded, as a ragged batch has a new number of tokens every step; a call of a new shape
# works it all out (prefill 25.9 us of host time, 12.6 with a plan).
_PLANS: dict = {}


def _layout(*tensors):
    return tuple((t.shape, t.stride(), t.dtype, t.get_device()) for t in tensors)


def _settings(window, sinks, scale, soft_cap):
    """The settings as plain numbers (a plan is found by their values)."""
    # (no sequence has more than 2^31 - 1 keys: the native arguments are 32 bits wide)
    return None if window is None else min(int(window), NO_WINDOW), min(int(sinks), NO_WINDOW), None if scale is None else float(scale), float(soft_cap)


def _remember(key, plan):
    if len(_PLANS) >= 4096:
        _PLANS.clear()
    _PLANS[key] = plan
    return plan


def _attention_args(q, k_cache, block_table, batch, splits, row_tiles, window, sinks, scale, soft_cap, shared):
    a = _lib.AttentionArgs()
    a.q_token, a.q_head = q.stride(0), q.stride(1)
    a.stride_block, a.stride_token, a.stride_head = k_cache.stride(0), k_cache.stride(1), k_cache.stride(2)
    a.tokens, a.B, a.Hq, a.Hkv, a.head_dim = q.shape[0], batch, q.shape[1], k_cache.shape[2], q.shape[2]
    a.page_size, a.max_blocks, a.blocks = k_cache.shape[1], block_table.shape[-1], k_cache.shape[0]
    a.splits, a.row_tiles, a.window, a.sinks = splits, row_tiles, window, sinks
    a.shared, a.dtype, a.scale, a.soft_cap = int(shared), _DTYPES[q.dtype], float(scale), float(soft_cap)
    return a


def _run_attention(template, q, k_cache, v_cache, table, starts, lens, out, parts, rows, status, handle):
    """``parts``: fp32 ``[splits * rows * (D + 1)]``, the partial results and behind them their LSE; None: none needed."""
    global launch_count
    a = _lib.AttentionArgs.from_buffer_copy(template)
    a.q, a.k_cache, a.v_cache = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    a.block_table, a.kv_lens = table.data_ptr(), lens.data_ptr()
    if starts is not None:
        a.q_starts = starts.data_ptr()
    if out is not None:
        a.out = out.data_ptr()
    if parts is not None:
        a.part_o = parts.data_ptr()
        a.part_lse = a.part_o + 4 * a.splits * rows * a.head_dim
    a.status, a.timeout_ns, a.stream = status, default_timeout_ns(), handle
    code = _lib.lib().tdist_attention(C.byref(a))
    if code:
        _lib.check(code, "tdist_attention")
    launch_count += 1
    return a


def _decode_call(template, q, k_cache, v_cache, table, lens, out, status, handle):
    """Arguments of the split decode kernel over windows, or with the partial results of another kernel."""
    a = _lib.DecodeArgs.from_buffer_copy(template)
    partial, counters = FD._Workspace.get(q.device, None, handle, a.B, a.Hq, a.Hkv, a.head_dim, a.splits)
    a.q, a.k_cache, a.v_cache = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    a.block_table, a.kv_lens, a.out = table.data_ptr(), lens.data_ptr(), out.data_ptr()
    a.partial, a.counters = partial.data_ptr(), counters.data_ptr()
    a.status, a.timeout_ns, a.stream = status, default_timeout_ns(), handle
    return a


def _run_decode(a):
    code = _lib.lib().tdist_flash_decode(C.byref(a))
    if code:
        _lib.check(code, "tdist_flash_decode")
    FD.launch_count += 1


def _decode_args(q, k_cache, block_table, window, sinks, scale, soft_cap, kv_split, priors=0):
    if not q.is_contiguous():
        raise ValueError("q must be contiguous")
    B, Hq, D = q.shape
    blocks, page, Hkv, _ = k_cache.shape
    a = _lib.DecodeArgs()
    a.B, a.Hq, a.Hkv, a.head_dim, a.page_size = B, Hq, Hkv, D, page
    a.max_blocks = block_table.shape[1]
    most = min(page * block_table.shape[1], window + sinks)
    a.splits = min(FD.choose_splits(B, Hq, Hkv, D, most, blocks * page, q.device) if kv_split <= 0 else kv_split, 256 - priors)
    a.stride_block, a.stride_token, a.stride_head = k_cache.stride(0), k_cache.stride(1), k_cache.stride(2)
    a.scale, a.soft_cap, a.dtype, a.world = float(scale), float(soft_cap), _DTYPES[q.dtype], 1
    a.window, a.sinks, a.priors, a.blocks = window, sinks, priors, blocks
    return a


def _status_ptr():
    st = global_status()
    return st.device_ptr if st is not None else None


@nvtx_range("tdist.gqa_fwd_window_decode")
def gqa_fwd_window_decode(q, k_cache, v_cache, kv_lens, block_table, window: Optional[int] = None, sinks: int = 0, scale=None,
                          soft_cap: float = 0.0, out: Optional[torch.Tensor] = None, kv_split: int = -1):
    """Decode attention of one query token per sequence over its last ``window`` keys and its first ``sinks``. Returns
    ``[B, Hq, D]`` in q's dtype; at most 16 query heads per kv head, q contiguous."""
    window, sinks, scale, soft_cap = _settings(window, sinks, scale, soft_cap)
    key = (gqa_fwd_window_decode, _layout(q, k_cache, v_cache, kv_lens, block_table), window, sinks, scale, soft_cap, kv_split)
    args = _PLANS.get(key)
    if args is None:
        B = q.shape[0]
        _check(q, k_cache, v_cache, window, sinks, soft_cap, (("kv_lens", kv_lens, (B,)), ("block_table", block_table, (B, None))), 16)
        factor = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
        if q.device.type != "cuda":
            return _stated(ref_window_attn(q, k_cache, v_cache, torch.arange(B + 1), kv_lens, block_table, window, sinks, factor, soft_cap), q, out)
        if B == 0:
            return _output(out, q)
        args = _remember(key, _decode_args(q, k_cache, block_table, NO_WINDOW if window is None else window, sinks, factor,
                                           soft_cap, kv_split))
    out = _output(out, q)
    table, lens = _int32(block_table), _int32(kv_lens)
    _run_decode(_decode_call(args, q, k_cache, v_cache, table, lens, out, _status_ptr(), stream_ptr(q.device)))
    return out


@nvtx_range("tdist.gqa_fwd_window_prefill")
def gqa_fwd_window_prefill(q, k_cache, v_cache, q_starts, kv_lens, block_table, window: Optional[int] = None, sinks: int = 0,
                           scale=None, soft_cap: float = 0.0, out: Optional[torch.Tensor] = None, kv_split: int = -1):
    """Attention of a ragged batch of query tokens, the last ones of their sequences. Returns ``[T, Hq, D]`` in q's dtype; at most 128
    query heads per kv head. q may be a view (part of a fused projection) with strides that are multiples of 8 elements; nothing is read
    back to the host."""
    window, sinks, scale, soft_cap = _settings(window, sinks, scale, soft_cap)
    key = (gqa_fwd_window_prefill, _layout(q, k_cache, v_cache, q_starts, kv_lens, block_table), window, sinks, scale, soft_cap, kv_split)
    args = _PLANS.get(key)
    if args is None:
        B = kv_lens.shape[0]
        _check(q, k_cache, v_cache, window, sinks, soft_cap,
               (("kv_lens", kv_lens, (B,)), ("q_starts", q_starts, (B + 1,)), ("block_table", block_table, (B, None))), 128)
        factor = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
        if q.device.type != "cuda":
            return _stated(ref_window_attn(q, k_cache, v_cache, q_starts, kv_lens, block_table, window, sinks, factor, soft_cap), q, out)
        T, Hq, D = q.shape
        if T == 0 or B == 0 or block_table.shape[1] == 0:
            return _output(out, q).zero_()
        most = NO_WINDOW if window is None else window
        tile = 128 // (Hq // k_cache.shape[2])
        each = -(-T // B)                                   # tokens of a sequence, where all have as many
        row_tiles = 2 if D <= 128 and each > tile else 1
        splits = kv_split
        if splits <= 0:
            ctas = B * -(-each // (tile * row_tiles)) * k_cache.shape[2]
            keys = min(block_table.shape[1] * k_cache.shape[1], most + sinks + tile * row_tiles)
            splits = _splits(ctas, keys, D, FD._sm_count(q.device))
        args = _remember(key, _attention_args(q, k_cache, block_table, B, splits, row_tiles, most, sinks, factor, soft_cap, False))
    out = _output(out, q)
    rows = args.tokens * args.Hq
    parts = torch.empty(args.splits * rows * (args.head_dim + 1), dtype=torch.float32, device=q.device) if args.splits > 1 else None
    _run_attention(args, q, k_cache, v_cache, _int32(block_table), _int32(q_starts), _int32(kv_lens), out, parts, rows, _status_ptr(),
                   stream_ptr(q.device))
    return out


@nvtx_range("tdist.gqa_fwd_shared_prefix_decode")
def gqa_fwd_shared_prefix_decode(q, k_cache, v_cache, prefix_len, prefix_table, kv_lens, block_table, scale=None, soft_cap: float = 0.0,
                                 out: Optional[torch.Tensor] = None, kv_split: int = -1):
    """Decode attention of one query token per sequence over a prefix that all share and the sequence's own keys. The prefix is in
    the pages ``prefix_table`` (``prefix_len`` keys; an integer tensor of one element on the device, or a number), the own keys in those of
    ``block_table`` (``kv_lens`` keys, which may be zero). Returns ``[B, Hq, D]`` in q's dtype; at most 16 query heads per kv head,
    q contiguous. ``kv_split``: parts of the prefix."""
    if not isinstance(prefix_len, torch.Tensor):
        prefix_len = torch.full((1,), int(prefix_len), dtype=torch.int32, device=q.device)
    _, _, scale, soft_cap = _settings(None, 0, scale, soft_cap)
    key = (gqa_fwd_shared_prefix_decode, _layout(q, k_cache, v_cache, prefix_len, prefix_table, kv_lens, block_table), scale, soft_cap, kv_split)
    plan = _PLANS.get(key)
    if plan is None:
        B = q.shape[0]
        _check(q, k_cache, v_cache, None, 0, soft_cap,
               (("prefix_len", prefix_len, (1,)), ("prefix_table", prefix_table, (None,)), ("kv_lens", kv_lens, (B,)), ("block_table", block_table, (B, None))),
               16)
        factor = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
        if q.device.type != "cuda":
            return _stated(ref_shared_prefix_attn(q, k_cache, v_cache, prefix_len, prefix_table, kv_lens, block_table, factor, soft_cap), q, out)
        _, Hq, D = q.shape
        if B == 0:
            return _output(out, q)
        first, splits = None, 0
        if prefix_table.shape[0] > 0:
            tile = 128 // (Hq // k_cache.shape[2])
            row_tiles = 2 if D <= 128 and B > tile else 1
            splits = kv_split
            if splits > 200:
                raise ValueError("kv_split must be at most 200")
            if splits <= 0:
                splits = _splits(-(-B // (tile * row_tiles)) * k_cache.shape[2], prefix_table.shape[0] * k_cache.shape[1], D, FD._sm_count(q.device))
            first = _attention_args(q, k_cache, prefix_table, 1, splits, row_tiles, NO_WINDOW, 0, factor, soft_cap, True)
        plan = _remember(key, (first, _decode_args(q, k_cache, block_table, NO_WINDOW, 0, factor, soft_cap, -1, splits)))
    first, second = plan
    out = _output(out, q)
    status, handle = _status_ptr(), stream_ptr(q.device)
    own_table, own_lens = _int32(block_table), _int32(kv_lens)
    own = _decode_call(second, q, k_cache, v_cache, own_table, own_lens, out, status, handle)
    if first is not None:
        rows = first.tokens * first.Hq
        parts = torch.empty(first.splits * rows * (first.head_dim + 1), dtype=torch.float32, device=q.device)
        prefix = _run_attention(first, q, k_cache, v_cache, _int32(prefix_table), None, _int32(prefix_len), None, parts, rows, status, handle)
        own.prior_o, own.prior_lse = prefix.part_o, prefix.part_lse
    _run_decode(own)
    return out
