"""A paged KV cache in 8 or 4 bits: quantised as it is written, read back, and attended to by single query tokens.

* ``create_quantized_kv_cache(blocks, page_size, kv_heads, head_dim, bits) -> QuantizedKVCache``
* ``kv_cache_write(cache, k[T,Hkv,D], v, slots[T])``: token t goes to place ``slots[t] % page_size`` of page ``slots[t] // page_size``
* ``kv_cache_read(cache, starts[B+1], kv_lens[B], block_table[B,max_blocks], rows, dtype) -> (k, v) [rows,Hkv,D]``: sequence b's keys are
  rows ``starts[b] .. starts[b] + kv_lens[b] - 1``; with starts that are multiples of a page size the rows are a paged cache again,
  which the prefill of :mod:`.paged_attention` reads
* ``gqa_fwd_quantized_decode(q[B,Hq,D], cache, kv_lens, block_table, window, sinks, scale, soft_cap) -> [B,Hq,D]``

The format, per row of D values (one token's key or value of one head):

* 8 bits: ``a = max(max|x|, 2^-100)``, ``scale = a / 127`` in fp32, ``code = 128 + rint(x (127 / a))``; value ``(code - 128) scale``
* 4 bits, for every 64 values: ``least`` the minimum rounded down to bf16, ``step = max((max - least) / 15, 2^-100)`` rounded up to bf16,
  ``code = rint((x - least) (1 / step))`` in 0..15; value ``least + step code``. Two codes per byte, the even index in the low half.

So a key and value of 128 dimensions take 264 and 144 bytes where bf16 takes 512. A row (64 values) that holds a NaN or an infinity is
stored with a scale of NaN: it reads as NaN, and so does the result of every query that sees it. A finite row reads as finite in the type that it was written in: what 4 bits put
beyond the type's largest number by up to half a step reads as that number. Codes are exact in every product; a result
differs from attention over the rows read back only by roundings: of the query to 16 bits (elements below 2^-6 of its largest in bf16, 2^-3 in fp16, by up to
1 / 32640 of the largest), of each key's weight times its value's scale to fp16 (2^-11 of itself, or 2^-30 of the largest such product of the head; fp16 results: a second number for
what is left), and of the result.

Slots must differ, as a server's pages do: of two tokens with one slot either's codes may stay beside the other's scale. Tokens whose slot is
no place of the cache (a negative one: padding) are left out. Lengths are cut to what the table has room for (at most 2^31 - 64 keys), and a page that the cache does not
have reads as zeros: nothing outside the tensors is touched.

CUDA tensors run ``csrc/kernels/quantized_cache.cu`` and ``quantized_decode.cu``, CPU tensors the plain statements. No call keeps
scratch memory: calls on any streams, captured or not, are independent.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Optional, Tuple

import torch

from .. import _lib
from ..utils.profile import nvtx_range
from . import flash_decode as FD
from . import paged_attention as PA

launch_count = 0
GROUP = 64            # values that share a pair of 4-bit scales
LEAST = 2.0 ** -100   # magnitudes below it count as it
MOST_KEYS = (1 << 31) - 64   # of a sequence: whole tiles of them are counted in 31 bits
_DTYPES = {torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16}


class QuantizedKVCache(NamedTuple):
    """Codes uint8 ``[blocks, page, Hkv, D]`` (8 bits) or ``[blocks, page, Hkv, D/2]`` (4 bits); scales fp32 ``[blocks, Hkv, page]`` or
    pairs of bf16 (step, least) ``[blocks, Hkv, page, D/64, 2]``: which one it is says the bits."""
    k: torch.Tensor
    v: torch.Tensor
    k_scales: torch.Tensor
    v_scales: torch.Tensor

    @property
    def bits(self) -> int:
        return 8 if self.k_scales.dim() == 3 else 4

    @property
    def head_dim(self) -> int:
        return self.k.shape[3] * (8 // self.bits)


def create_quantized_kv_cache(blocks: int, page_size: int, kv_heads: int, head_dim: int, bits: int = 8, device="cuda") -> QuantizedKVCache:
    """A cache of zeros."""
    if bits not in (8, 4):
        raise ValueError("a quantised cache has 8 or 4 bits")
    if head_dim < GROUP or head_dim % GROUP:
        raise ValueError(f"head_dim must be a multiple of {GROUP}")
    codes = [torch.full((blocks, page_size, kv_heads, head_dim * bits // 8), 128 if bits == 8 else 0, dtype=torch.uint8, device=device) for _ in range(2)]
    shape = (blocks, kv_heads, page_size) + (() if bits == 8 else (head_dim // GROUP, 2))
    scales = [torch.zeros(shape, dtype=torch.float32 if bits == 8 else torch.bfloat16, device=device) for _ in range(2)]
    return QuantizedKVCache(*codes, *scales)


# ---------------------------------------------------------------------------- plain statements
def quotient(a, b) -> torch.Tensor:
    """a / b rounded once, one of them a tensor (with a number on either side torch may multiply by a rounded reciprocal)."""
    t = a if isinstance(a, torch.Tensor) else b
    return torch.div(a if t is a else torch.full_like(t, a), b if t is b else torch.full_like(t, b))


def _bf16_down(x: torch.Tensor) -> torch.Tensor:
    """The largest bf16 that is not above x (fp32), as fp32."""
    b = x.to(torch.bfloat16)
    return torch.where(b.float() > x, torch.nextafter(b, torch.full_like(b, -math.inf)), b).float()


def ref_quantize_rows(x: torch.Tensor, bits: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows ``[..., D]`` -> codes and scales ``[...]`` / pairs ``[..., D/64, 2]``."""
    x = x.float()
    if bits == 8:
        most = x.abs().amax(-1, keepdim=True)
        good = most < math.inf   # (false for NaN)
        most = torch.where(good, most, 1.0).clamp_min(LEAST)
        code = torch.where(good, torch.round(x * quotient(127.0, most)), 0.0) + 128.0
        return code.to(torch.uint8), torch.where(good, quotient(most, 127.0), math.nan).squeeze(-1)
    g = x.unflatten(-1, (-1, GROUP))
    good = g.abs().amax(-1, keepdim=True) < math.inf
    g = torch.where(good, g, 0.0)
    least, most = _bf16_down(g.amin(-1, keepdim=True)), g.amax(-1, keepdim=True)
    half = torch.where((most - least).isinf(), 0.5, 1.0)   # of a range beyond fp32's largest: differences of halves
    step = -_bf16_down(-(quotient(most * half - least * half, 15.0) / half).clamp_min(LEAST))
    code = torch.round((g * half - least * half) * (quotient(1.0, step) / half)).clamp(0.0, 15.0).to(torch.uint8).flatten(-2)
    pairs = torch.where(good, torch.cat([step, least], -1), math.nan)
    return code[..., 0::2] | (code[..., 1::2] << 4), pairs.to(torch.bfloat16)


def ref_dequantize_rows(codes: torch.Tensor, scales: torch.Tensor, bits: int, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Rows of codes and scales. 4 bits: a value beyond the type's largest number by no more than half a step is that number (a number that
    was not beyond may come to lie there by its rounding to a code and the pair's rounding outwards)."""
    if bits == 8:
        return ((codes.float() - 128.0) * scales.unsqueeze(-1)).to(dtype)
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double().unflatten(-1, (-1, GROUP))
    step, least = scales.double()[..., 0:1], scales.double()[..., 1:2]
    v, most = c * step + least, torch.finfo(dtype).max
    near = (v.abs() > most) & (v.abs() - step / 2 <= most)
    return torch.where(near, most * v.sign(), v).float().to(dtype).flatten(-2)


def ref_kv_cache_write(cache: QuantizedKVCache, k, v, slots) -> None:
    blocks, page = cache.k.shape[:2]
    kept = (slots >= 0) & (slots < blocks * page)
    at = slots[kept].long()
    for x, codes, scales in ((k, cache.k, cache.k_scales), (v, cache.v, cache.v_scales)):
        c, s = ref_quantize_rows(x[kept], cache.bits)
        codes[at // page, at % page] = c
        scales.transpose(1, 2)[at // page, at % page] = s


def _rows_of(cache: QuantizedKVCache, table, at, dtype=torch.float32):
    """k and v of the positions ``at`` of one sequence; zeros for pages that the cache does not have."""
    blocks, page = cache.k.shape[:2]
    pages, rows = table[at // page].long(), at % page
    there = (pages >= 0) & (pages < blocks)
    pages = torch.where(there, pages, 0)
    out = []
    for codes, scales in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)):
        x = ref_dequantize_rows(codes[pages, rows], scales.transpose(1, 2)[pages, rows], cache.bits, dtype)
        out.append(torch.where(there.view(-1, 1, 1), x, 0.0))
    return out


def _limits(cache, block_table, kv_lens):
    """Lengths on the host, cut to the table and to what the kernels count."""
    room = min(block_table.shape[1] * cache.k.shape[1], MOST_KEYS) if cache.k.shape[0] else 0
    return [min(max(int(n), 0), room) for n in kv_lens]


def ref_kv_cache_read(cache: QuantizedKVCache, starts, kv_lens, block_table, rows: int, dtype=torch.bfloat16):
    out = [torch.zeros((rows, cache.k.shape[2], cache.head_dim), dtype=dtype, device=cache.k.device) for _ in range(2)]
    for b, n in enumerate(_limits(cache, block_table, kv_lens)):
        r0 = int(starts[b])
        n = min(n, int(starts[b + 1]) - r0, rows - r0)
        if n > 0 and r0 >= 0:
            for o, x in zip(out, _rows_of(cache, block_table[b], torch.arange(n, device=cache.k.device), dtype)):
                o[r0:r0 + n] = x
    return out[0], out[1]


def ref_quantized_decode(q, cache: QuantizedKVCache, kv_lens, block_table, window=None, sinks: int = 0, scale=None, soft_cap: float = 0.0):
    """fp32 attention of the rows read back."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float32, device=q.device)
    for b, n in enumerate(_limits(cache, block_table, kv_lens)):
        lo = 0 if window is None else max(0, n - window)
        at = torch.cat([torch.arange(0, min(sinks, lo)), torch.arange(lo, n)]).to(q.device)
        if at.numel():
            k, v = _rows_of(cache, block_table[b], at)
            out[b:b + 1] = PA._attend(q[b:b + 1], k, v, torch.ones((1, at.numel()), dtype=torch.bool, device=q.device), scale, soft_cap)
    return out


# ---------------------------------------------------------------------------- calls
# Native arguments but for the pointers, and the checks that led there, by shapes, strides, types and settings (never by addresses or contents).
_PLANS: dict = {}


def _remember(key, plan):
    if len(_PLANS) >= 4096:
        _PLANS.clear()
    _PLANS[key] = plan
    return plan


def _check_cache(cache: QuantizedKVCache):
    k, v, ks, vs = cache
    if k.dim() != 4 or ks.dim() not in (3, 5):
        raise ValueError("codes must be [blocks, page, Hkv, D] (4 bits: D / 2), scales [blocks, Hkv, page] (4 bits: [blocks, Hkv, page, D / 64, 2])")
    bits, D = cache.bits, cache.head_dim
    blocks, page, Hkv, _ = k.shape
    want = (blocks, Hkv, page) + (() if bits == 8 else (D // GROUP, 2))
    if v.shape != k.shape or ks.shape != want or vs.shape != want:
        raise ValueError(f"codes {tuple(k.shape)} and {tuple(v.shape)} need scales {want}, got {tuple(ks.shape)} and {tuple(vs.shape)}")
    if page < 1 or Hkv < 1 or D < GROUP or D % GROUP:
        raise ValueError(f"pages and heads must not be empty, head_dim a multiple of {GROUP}")
    if blocks * page >= 1 << 31:
        raise ValueError("a cache has at most 2^31 - 1 places")
    if k.dtype != torch.uint8 or v.dtype != torch.uint8 or any(s.dtype != (torch.float32 if bits == 8 else torch.bfloat16) for s in (ks, vs)):
        raise TypeError("codes are uint8; scales fp32 (8 bits) or bf16 (4 bits)")
    if any(t.device != k.device for t in cache):
        raise ValueError("codes and scales must be on one device")
    if k.device.type != "cuda":
        return
    if D not in (64, 128, 256):
        raise ValueError("head_dim must be 64, 128 or 256")
    if v.stride() != k.stride() or vs.stride() != ks.stride():
        raise ValueError("the codes of k and v need equal strides, and so do their scales")
    inner = bits == 8 or (ks.stride(4) == 1 and (ks.shape[3] == 1 or ks.stride(3) == 2))
    if k.stride(3) != 1 or not inner:
        raise ValueError("the codes of a row, and its scales, must be contiguous")


def _check_ints(device, ints):
    for name, t, shape in ints:
        if t.dim() != len(shape) or any(s is not None and s != n for s, n in zip(shape, t.shape)):
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {['any' if s is None else s for s in shape]}")
        if t.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"{name} must hold integers (int32 or int64)")
        if any(n >= 1 << 31 for n in t.shape):
            raise ValueError(f"{name} has shape {tuple(t.shape)}: sizes are counted in 31 bits")
        if t.device != device:
            raise ValueError(f"{name} must be on the cache's device")


def _cache_args(cache: QuantizedKVCache, dtype) -> "_lib.QuantCacheArgs":
    a = _lib.QuantCacheArgs()
    k, ks = cache.k, cache.k_scales
    a.code_block, a.code_token, a.code_head = k.stride(0), k.stride(1), k.stride(2)
    size = ks.element_size()
    a.scale_block, a.scale_head, a.scale_token = ks.stride(0) * size, ks.stride(1) * size, ks.stride(2) * size
    a.blocks, a.page_size, a.Hkv, a.head_dim, a.bits = k.shape[0], k.shape[1], k.shape[2], cache.head_dim, cache.bits
    a.dtype = _DTYPES[dtype]
    return a


def _of(t: torch.Tensor):
    return t.shape, t.stride(), t.dtype, t.get_device()


def _layout(cache: QuantizedKVCache):
    """What a plan is found by, the device last: codes and scales of k and v have to be alike, so theirs are compared and k's told."""
    k, v, ks, vs = cache
    codes, scales = _of(k), _of(ks)
    return _of(v) == codes and _of(vs) == scales, codes, scales, codes[3]


def _plain(*ints):
    return all(t.dtype == torch.int32 and t.is_contiguous() for t in ints)


def _point(a, cache: QuantizedKVCache, index: int):
    k, v, ks, vs = cache
    a.k_codes, a.v_codes, a.k_scales, a.v_scales = k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr()
    a.stream = torch._C._cuda_getCurrentRawStream(index)


def _launch(fn, a, index: int, what: str):
    """The native call with device ``index`` as the current one."""
    global launch_count
    if index == torch._C._cuda_getDevice():
        code = fn(C.byref(a))
    else:
        with torch.cuda.device(index):
            code = fn(C.byref(a))
    if code:
        _lib.check(code, what)
    launch_count += 1


@nvtx_range("tdist.kv_cache_write")
def kv_cache_write(cache: QuantizedKVCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantises ``k, v [T, Hkv, D]`` (bf16 or fp16; views of a fused projection are read in place) into their places ``slots [T]``.
    What the slots do not name keeps its bytes."""
    layout = _layout(cache)
    key = (kv_cache_write, layout, _of(k), _of(v), _of(slots))
    plan = _PLANS.get(key)
    if plan is None:
        _check_cache(cache)
        want = (slots.shape[0] if slots.dim() else 0, cache.k.shape[2], cache.head_dim)
        if k.shape != want or v.shape != want:
            raise ValueError(f"k and v must be [T, Hkv, D] = {want}, got {tuple(k.shape)} and {tuple(v.shape)}")
        _check_ints(cache.k.device, (("slots", slots, (None,)),))
        if k.dtype not in _DTYPES or v.dtype != k.dtype:
            raise TypeError("k and v must share one of bf16 / fp16")
        if k.device != cache.k.device or v.device != cache.k.device:
            raise ValueError("k and v must be on the cache's device")
        if cache.k.device.type != "cuda":
            ref_kv_cache_write(cache, k, v, slots)
            return
        args = _cache_args(cache, k.dtype)
        args.rows = k.shape[0]
        args.k_token, args.k_head, args.v_token, args.v_head = 2 * k.stride(0), 2 * k.stride(1), 2 * v.stride(0), 2 * v.stride(1)
        # rows are loaded by 16 bytes
        plan = _remember(key, (args, _plain(slots), all(x.stride(2) == 1 and x.stride(0) % 8 == 0 and x.stride(1) % 8 == 0 for x in (k, v))))
    args, plain, loads = plan
    if args.rows == 0 or args.blocks == 0:
        return
    a = _lib.QuantCacheArgs.from_buffer_copy(args)
    if not plain:
        # no place of the cache is beyond 32 bits, but a slot may be
        slots = slots.clamp(-1, 0x7FFFFFFF).to(torch.int32).contiguous()
    if not loads or (k.data_ptr() | v.data_ptr()) % 16:
        k, v = (x.clone(memory_format=torch.contiguous_format) for x in (k, v))
        a.k_token = a.v_token = 2 * a.Hkv * a.head_dim
        a.k_head = a.v_head = 2 * a.head_dim
    a.k, a.v, a.slots = k.data_ptr(), v.data_ptr(), slots.data_ptr()
    _point(a, cache, layout[-1])
    _launch(_lib.lib().tdist_quant_cache_write, a, layout[-1], "tdist_quant_cache_write")


def _int32(t):
    return (t if t.dtype == torch.int32 else t.clamp(-0x80000000, 0x7FFFFFFF).to(torch.int32)).contiguous()


@nvtx_range("tdist.kv_cache_read")
def kv_cache_read(cache: QuantizedKVCache, starts: torch.Tensor, kv_lens: torch.Tensor, block_table: torch.Tensor, rows: int,
                  dtype: torch.dtype = torch.bfloat16, out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of a batch as rows of ``dtype`` (bf16 or fp16): sequence b's first ``kv_lens[b]`` keys from row ``starts[b]`` on, at most
    up to ``starts[b + 1]`` (``starts`` must not decrease; a sequence with a negative one is not read). Returns ``(k, v)``, each ``[rows, Hkv, D]`` (``out``, if given); rows of no
    sequence are zeros."""
    rows = int(rows)
    given = () if out is None else tuple(out)
    layout = _layout(cache)
    key = (kv_cache_read, layout, _of(starts), _of(kv_lens), _of(block_table), rows, dtype, given and tuple(map(_of, given)))
    plan = _PLANS.get(key)
    if plan is None:
        _check_cache(cache)
        if rows < 0 or rows >= 1 << 31:
            raise ValueError("rows must lie in [0, 2^31)")
        if dtype not in _DTYPES:
            raise TypeError("rows are read as bf16 or fp16")
        B = kv_lens.shape[0] if kv_lens.dim() else 0
        _check_ints(cache.k.device, (("kv_lens", kv_lens, (B,)), ("starts", starts, (B + 1,)), ("block_table", block_table, (B, None))))
        shape = (rows, cache.k.shape[2], cache.head_dim)
        if out is not None and (len(given) != 2 or any(o.shape != shape or o.dtype != dtype or o.device != cache.k.device or not o.is_contiguous() for o in given)):
            raise ValueError(f"out must be two contiguous tensors {shape} of {dtype} on the cache's device")
        if cache.k.device.type != "cuda":
            ref = ref_kv_cache_read(cache, starts, kv_lens, block_table, rows, dtype)
            return ref if out is None else (given[0].copy_(ref[0]), given[1].copy_(ref[1]))
        args = _cache_args(cache, dtype)
        args.rows, args.B, args.max_blocks = rows, B, block_table.shape[1]
        plan = _remember(key, (args, _plain(starts, kv_lens, block_table)))
    args, plain = plan
    if out is None:
        k = cache.k.new_empty(rows, args.Hkv, args.head_dim, dtype=dtype)
        v = torch.empty_like(k)
    else:
        k, v = given
    if rows == 0:
        return k, v
    a = _lib.QuantCacheArgs.from_buffer_copy(args)
    if not plain:
        starts, kv_lens, block_table = _int32(starts), _int32(kv_lens), _int32(block_table)
    a.starts, a.lens, a.table = starts.data_ptr(), kv_lens.data_ptr(), block_table.data_ptr()
    a.k_out, a.v_out = k.data_ptr(), v.data_ptr()
    _point(a, cache, layout[-1])
    _launch(_lib.lib().tdist_quant_cache_read, a, layout[-1], "tdist_quant_cache_read")
    return k, v


MOST_SHARED = 511   # sequences of a call whose keys are dealt out in shares


def _decode_parts(B: int, per_b: int, most: int, table_keys: int, asked: int, slots: int, wide: bool):
    """(splits, shares) of a decode over at most ``most`` keys per sequence, ``per_b`` segments side by side for a sequence's heads; the machine
    has room for ``slots`` large CTAs (``wide``: one per SM, otherwise two). CTAs per segment; or 0 and the CTAs that take equal shares of
    all sequences; or 0, 0: a small CTA per segment.

    Small CTAs leave room for three (wide: two) times as many: a short segment is mostly latency and the meeting of its warps' sums (8 bits, 4 query
    heads on each of 8 kv heads of 128: 256 sequences of 512 keys 75.4 us with large CTAs, 58.2 with small ones, of 128 keys 43.1 and 22.7; 24 sequences
    of 512 keys 10.3 and 11.5; wide, 6 query heads on one of 256, 500 sequences of 1024 keys 66.7 and 51.7, of 4096 ones 188 and 165, as shares 178; 16 on
    one of 128, 300 of 1024 keys 49.3 and 40.0, as shares 40.6, of 4096 ones 104 and 107, as shares 81). A cluster's 8
    parts merge without a second kernel (one sequence, 4096 keys 10.4 us and 12.7 as shares, 8192 keys 13.4 and 13.7)."""
    may_share = B <= MOST_SHARED and B * (-(-table_keys // 16) + 2) < 1 << 31
    segments = B * per_b
    if asked == 0:
        return 0, 0
    if asked > 0:
        return (asked, 0) if asked <= 8 else ((0, max(1, min(slots // per_b, B * asked))) if may_share else (8, 0))
    if most <= (256 if segments <= slots else 4096 if wide else min(2048, 256 + segments)):
        return 0, 0
    splits = max(1, min(slots // max(1, segments), -(-most // 256)))
    if may_share and ((splits > 8 and most > 8 * 768) or (most >= 1024 and segments * most > slots * 2048)):
        return 0, max(1, slots // per_b)
    return min(splits, 8), 0


@nvtx_range("tdist.gqa_fwd_quantized_decode")
def gqa_fwd_quantized_decode(q: torch.Tensor, cache: QuantizedKVCache, kv_lens: torch.Tensor, block_table: torch.Tensor,
                             window: Optional[int] = None, sinks: int = 0, scale=None, soft_cap: float = 0.0,
                             out: Optional[torch.Tensor] = None, kv_split: int = -1) -> torch.Tensor:
    """Decode attention of one query token per sequence over a quantised cache: the query of a sequence of n keys sees key j if
    j >= n - window or j < sinks (``window=None``: all keys). ``q [B, Hq, D]`` bf16 or fp16, contiguous; returns its shape and type. A
    query that sees no key (or none whose score is above -inf) gives zeros. Pages without a visible key are not read. ``kv_split``: parts of a
    sequence's keys, up to 8; more: equal shares of all sequences' keys, as many as fit the machine; 0: one part by few warps, for many short
    sequences; -1: chosen by sizes."""
    window, sinks, scale, soft_cap = PA._settings(window, sinks, scale, soft_cap)
    layout = _layout(cache)
    key = (gqa_fwd_quantized_decode, layout, _of(q), _of(kv_lens), _of(block_table), window, sinks, scale, soft_cap, kv_split)
    plan = _PLANS.get(key)
    if plan is None:
        _check_cache(cache)
        if q.dim() != 3 or q.shape[2] != cache.head_dim:
            raise ValueError("q must be [B, Hq, D] with the cache's head_dim")
        B, Hq, D = q.shape
        Hkv = cache.k.shape[2]
        if Hq < 1 or Hq % Hkv:
            raise ValueError("the query heads must be a multiple of the kv heads")
        if window is not None and window < 1:
            raise ValueError("the window must be at least 1 (None: no limit)")
        if sinks < 0 or not soft_cap >= 0:
            raise ValueError("sinks and soft_cap must not be negative")
        if q.device != cache.k.device:
            raise ValueError("q must be on the cache's device")
        _check_ints(q.device, (("kv_lens", kv_lens, (B,)), ("block_table", block_table, (B, None))))
        factor = 1.0 / math.sqrt(D) if scale is None else scale
        if q.device.type != "cuda":
            return PA._stated(ref_quantized_decode(q, cache, kv_lens, block_table, window, sinks, factor, soft_cap), q, out)
        if q.dtype not in _DTYPES:
            raise TypeError("q must be bf16 or fp16")
        if not q.is_contiguous():
            raise ValueError("q must be contiguous")
        args = _lib.QuantDecodeArgs()
        args.cache = _cache_args(cache, q.dtype)
        args.cache.B, args.cache.max_blocks = B, block_table.shape[1]
        args.Hq, args.window, args.sinks = Hq, PA.NO_WINDOW if window is None else window, sinks
        args.scale, args.soft_cap = factor, soft_cap
        two = Hq // Hkv > 8 and D != 256   # tiles of 8 query heads per segment
        wide = two or D == 256
        most = min(cache.k.shape[1] * block_table.shape[1], args.window + sinks)
        per_b = Hkv * -(-(Hq // Hkv) // (16 if two else 8))
        args.splits, args.shares = _decode_parts(B, per_b, most, cache.k.shape[1] * block_table.shape[1], kv_split,
                                                 (1 if wide else 2) * FD._sm_count(q.device), wide)
        # scratch of the shares: per CTA four words, and two times the sums of its heads
        args.scratch = args.shares * per_b * (4 + 2 * (16 if two else 8) * (D + 2))
        plan = _remember(key, (args, _plain(kv_lens, block_table)))
    args, plain = plan
    out = torch.empty_like(q) if out is None else PA._output(out, q)
    a = _lib.QuantDecodeArgs.from_buffer_copy(args)
    if a.cache.B == 0:
        return out
    if not plain:
        kv_lens, block_table = _int32(kv_lens), _int32(block_table)
    c = a.cache
    _point(c, cache, layout[-1])
    c.lens, c.table = kv_lens.data_ptr(), block_table.data_ptr()
    if q.data_ptr() % 16:
        q = q.clone()
    a.q, a.out = q.data_ptr(), out.data_ptr()
    if a.shares:
        part = torch.empty(a.scratch, dtype=torch.float32, device=q.device)
        a.part = part.data_ptr()
    _launch(_lib.lib().tdist_quant_decode, a, layout[-1], "tdist_quant_decode")
    return out
