"""Paged key/value cache: rotated append, and attention over it.

The steps of a decoder layer between the switched QKV projection and the
switched output projection:

    slots, positions = cache_slots(page_table, kv_lens, page_size, num_pages, cu_seqlens)   # once per step
    q = append_kv_(q, k, v, k_cache, v_cache, slots, positions, cos_sin)                    # per layer
    o = paged_attention(q, k_cache, v_cache, page_table, kv_lens, cu_seqlens)

A cache is [num_pages, kv_heads, page_size, head_dim] with any order of its first
three dimensions in memory (``allocate_cache`` keeps a head's rows of a page
side by side).  Sequence s has its token j in row j % page_size of page
page_table[s, j // page_size]; kv_lens[s] counts its tokens, those of the call
among them.  An aLoRA adapter that switches on mid-sequence attends over the
base model's cached prefix this way: its few invocation tokens are a chunk of
queries (``cu_seqlens``) over a long cache.

A cache may be quantised (``allocate_quantized_cache``, ``QuantizedCache``): e4m3
values and a power of two for each row, half the bytes of bfloat16.  The calls are
the same; ``read_kv`` gives rows back.

Everything is launched on torch's current stream without host synchronisation;
bfloat16 or float32.  No gradients are computed: inputs that autograd tracks are
refused where gradients are enabled, and those with a forward-mode tangent everywhere.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import _lib

_INT32 = 2 ** 31 - 1        # what the library's 32-bit arguments hold; ctypes cuts larger values silently
_DTYPES = {torch.bfloat16: _lib.GS_DTYPE_BF16, torch.float32: _lib.GS_DTYPE_FP32}


def allocate_cache(num_pages: int, kv_heads: int, page_size: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
                   device="cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """A key and a value cache [num_pages, kv_heads, page_size, head_dim].

    A head's rows of a page lie side by side, so a page of 16 rows of 128 bf16
    values is one run of 4 KB.  The contents are not initialised: rows are read
    only once they were stored.
    """
    shape = (num_pages, kv_heads, page_size, head_dim)
    return torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device)


class QuantizedCache(NamedTuple):
    """A key or a value cache of 8-bit rows: a row of ``values`` times its power of two in ``scales``.

    values [num_pages, kv_heads, page_size, head_dim] float8_e4m3fn
    scales [num_pages, kv_heads, page_size] float8_e8m0fnu, a head's scales of a page side by side

    ``append_kv_`` takes the smallest power of two (2^-126 at least) that keeps a row's
    largest magnitude within 448, the largest e4m3 value, and rounds to nearest, ties to
    even: a value is off by at most 2^-4 of itself, or 2^-10 of its scale where that is
    more, and a finite one stays finite (magnitudes past 1.875 2^127 are kept as that).
    What is not finite becomes NaN, and the row's other values are kept.  A scale's byte
    is the power of two's exponent + 127: 0 is 2^-127 and 255 NaN, and ``append_kv_``
    writes neither.
    """

    values: torch.Tensor
    scales: torch.Tensor


def allocate_quantized_cache(num_pages: int, kv_heads: int, page_size: int, head_dim: int,
                             device="cuda") -> tuple[QuantizedCache, QuantizedCache]:
    """A key and a value cache of e4m3 rows, laid out as ``allocate_cache`` has them; not initialised.

    ``append_kv_`` and ``read_kv`` take any page_size and a head_dim up to 512; ``paged_attention`` takes pages of a
    multiple of 8 rows and a head_dim that is a multiple of 16 up to 256.
    """
    one = lambda: QuantizedCache(  # noqa: E731
        torch.empty((num_pages, kv_heads, page_size, head_dim), dtype=torch.float8_e4m3fn, device=device),
        torch.empty((num_pages, kv_heads, page_size), dtype=torch.float8_e8m0fnu, device=device))
    return one(), one()


def rope_table(max_pos: int, rot_dim: int, theta: float = 10000.0, device="cuda",
               inv_freq: torch.Tensor | None = None, scaling: float = 1.0) -> torch.Tensor:
    """The rotation table [max_pos, rot_dim] fp32: per position rot_dim/2 cosines, then rot_dim/2 sines.

    Angles are position * theta^(-2j / rot_dim) (or * ``inv_freq`` [rot_dim/2]),
    computed in 64 bits: a 32-bit product at position 10^6 is off by 0.06.
    ``scaling`` multiplies cosines and sines (an attention factor).
    """
    if rot_dim % 2 or rot_dim <= 0:
        raise ValueError(f"rope_table: rot_dim={rot_dim} must be even and positive")
    if inv_freq is None:
        inv_freq = theta ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device) / rot_dim)
    elif inv_freq.numel() != rot_dim // 2:
        raise ValueError(f"rope_table: inv_freq has {inv_freq.numel()} entries, rot_dim={rot_dim} needs {rot_dim // 2}")
    angle = torch.arange(max_pos, dtype=torch.float64, device=device)[:, None] * inv_freq.to(device, torch.float64)[None, :]
    return (torch.cat([angle.cos(), angle.sin()], dim=1) * scaling).float()


# ---------------------------------------------------------------------------
# Checks
# ---------------------------------------------------------------------------
def _heads3(who: str, name: str, t: torch.Tensor, tokens: int | None, dtype) -> torch.Tensor:
    if t.dim() != 3 or t.dtype != dtype or (tokens is not None and t.shape[0] != tokens):
        raise ValueError(f"{who}: {name} must be a {dtype} tensor [{'tokens' if tokens is None else tokens}, heads, "
                         f"head_dim], got {t.dtype} {tuple(t.shape)}")
    if t.stride(2) != 1 and t.shape[2] > 1:
        raise ValueError(f"{who}: {name}'s head dimension must be contiguous (strides {t.stride()})")
    if max(t.shape[1:]) > _INT32:
        raise ValueError(f"{who}: {name} has {t.shape[1]} heads of {t.shape[2]} (2^31 - 1 at most)")
    return t


def _caches(who: str, k_cache: torch.Tensor, v_cache: torch.Tensor, dtype, kv_heads, head_dim: int):
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        if c.dim() != 4 or c.dtype != dtype or c.shape != k_cache.shape or c.shape[3] != head_dim or \
                (kv_heads is not None and c.shape[1] != kv_heads):
            raise ValueError(f"{who}: {name} must be a {dtype} tensor [pages, kv_heads, page_size, {head_dim}], "
                             f"both caches alike, got {c.dtype} {tuple(c.shape)}")
        if c.stride(3) != 1 and head_dim > 1:
            raise ValueError(f"{who}: {name}'s head dimension must be contiguous (strides {c.stride()})")
    if k_cache.shape[0] == 0 or not 0 < k_cache.shape[2] <= _INT32 or k_cache.shape[1] > _INT32:
        raise ValueError(f"{who}: {k_cache.shape[0]} pages of {k_cache.shape[2]} rows and {k_cache.shape[1]} heads "
                         "(1 .. 2^31 - 1)")


def _scales(who: str, k_scales: torch.Tensor, v_scales: torch.Tensor, values: torch.Tensor):
    for name, t in (("k_cache", k_scales), ("v_cache", v_scales)):
        if t.dtype != torch.float8_e8m0fnu or t.shape != values.shape[:3]:
            raise ValueError(f"{who}: {name}'s scales must be a float8_e8m0fnu tensor {tuple(values.shape[:3])}, got "
                             f"{t.dtype} {tuple(t.shape)}")
        if t.stride(2) != 1 and t.shape[2] > 1:
            raise ValueError(f"{who}: {name}'s scales of a page must lie side by side (strides {t.stride()})")


def _parts(who: str, k_cache, v_cache):
    """``(k values, v values, k scales, v scales)``; no scales for a cache that is not quantised."""
    if isinstance(k_cache, QuantizedCache) != isinstance(v_cache, QuantizedCache):
        raise ValueError(f"{who}: one cache is quantised, the other is not")
    if isinstance(k_cache, QuantizedCache):
        return k_cache.values, v_cache.values, k_cache.scales, v_cache.scales
    return k_cache, v_cache, None, None


def _on_gpu(who: str, device: torch.device, *ts) -> None:
    if device.type != "cuda":
        raise ValueError(f"{who}: tensors must live on the GPU")
    for t in ts:
        if t is not None and t.device != device:
            raise ValueError(f"{who}: tensors must live on one GPU ({t.device} beside {device})")


def _ints(who: str, name: str, t: torch.Tensor, dtype, shape=None) -> torch.Tensor:
    if t.dtype != dtype or (shape is not None and tuple(t.shape) != tuple(shape)) or not t.is_contiguous():
        raise ValueError(f"{who}: {name} must be a contiguous {dtype} tensor"
                         f"{'' if shape is None else ' ' + str(tuple(shape))}, got {t.dtype} {tuple(t.shape)}")
    return t


def _table(who: str, page_table: torch.Tensor, seqs: int) -> torch.Tensor:
    if page_table.dim() != 2 or page_table.dtype != torch.int32 or page_table.shape[0] != seqs or \
            (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise ValueError(f"{who}: page_table must be an int32 tensor [{seqs}, max_pages] with contiguous rows, got "
                         f"{page_table.dtype} {tuple(page_table.shape)}")
    return page_table


def _table_ld(page_table: torch.Tensor) -> int:
    return page_table.stride(0) if page_table.shape[0] > 1 else max(page_table.stride(0), page_table.shape[1])


# What a call's checks found, by the shapes, strides, types and devices of its
# tensors (never by their addresses): a serving loop's calls repeat a few, and the
# checks take longer than a small call's kernel (9 of 15 us).
_append_plans: dict = {}
_rows_plans: dict = {}
_read_plans: dict = {}
_attention_plans: dict = {}
_PLAN_CAP = 4096


def _keep(plans: dict, key, plan):
    if len(plans) >= _PLAN_CAP:            # batch sizes vary per step: keep it bounded
        plans.clear()
    plans[key] = plan
    return plan


# ---------------------------------------------------------------------------
# Append
# ---------------------------------------------------------------------------
def cache_slots(page_table: torch.Tensor, kv_lens: torch.Tensor, page_size: int, num_pages: int,
                cu_seqlens: torch.Tensor | None = None,
                num_tokens: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(slots, positions)`` int64 [num_tokens] of a batch's tokens, once per step for every layer.

    Row i of sequence s's n rows is its token p = kv_lens[s] - n + i: the slot is
    page_table[s, p // page_size] * page_size + p % page_size, -1 where there is
    none (p < 0: a padding row).  ``cu_seqlens`` None: one row per sequence;
    otherwise ``num_tokens`` is the packed batch's row count.
    """
    who = "cache_slots"
    if _lib.elsewhere(kv_lens.device):
        with torch.cuda.device(kv_lens.device):
            return cache_slots(page_table, kv_lens, page_size, num_pages, cu_seqlens, num_tokens)
    B = kv_lens.shape[0]
    _on_gpu(who, kv_lens.device, page_table, cu_seqlens)
    _ints(who, "kv_lens", kv_lens, torch.int32, (B,))
    _table(who, page_table, B)
    if cu_seqlens is not None:
        _ints(who, "cu_seqlens", cu_seqlens, torch.int32, (B + 1,))
        if num_tokens is None:
            raise ValueError("cache_slots: cu_seqlens needs num_tokens (reading it would synchronise)")
    elif num_tokens is None:
        num_tokens = B
    elif num_tokens != B:
        raise ValueError(f"cache_slots: num_tokens={num_tokens} of {B} sequences without cu_seqlens")
    if not 0 < page_size <= _INT32:
        raise ValueError(f"cache_slots: page_size={page_size}")
    slots = torch.empty(num_tokens, dtype=torch.int64, device=kv_lens.device)
    positions = torch.empty(num_tokens, dtype=torch.int64, device=kv_lens.device)
    _lib.call("gs_cache_slots", page_table.data_ptr(), _table_ld(page_table), page_table.shape[1], int(num_pages),
              int(page_size), kv_lens.data_ptr(), _lib.ptr(cu_seqlens), B, int(num_tokens), slots.data_ptr(),
              positions.data_ptr(), _lib.stream_ptr(kv_lens.device))
    return slots, positions


def append_kv_(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, k_cache, v_cache,
               slots: torch.Tensor, positions: torch.Tensor | None = None, cos_sin: torch.Tensor | None = None,
               q_out: torch.Tensor | None = None, interleaved: bool = False, q_norm: torch.Tensor | None = None,
               k_norm: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor | None:
    """Rotate q and k by their positions, store k and v into the cache; returns the rotated q.

    q [T, heads, D], k and v [T, kv_heads, D]: views with contiguous head rows,
    such as slices of the QKV projection's output
    k_cache, v_cache: tensors of their type, or both ``QuantizedCache``
    slots     [T] int64: page * page_size + row; one outside the pool (-1) stores
              nothing (padding rows).  No two tokens may share a slot.
    positions [T] int64 and cos_sin [max_pos, R] fp32 (``rope_table``): the first R
              columns of a head are rotated as pairs (j, j + R/2), or (2j, 2j + 1)
              with ``interleaved``, the others copied.  cos_sin None: no rotation.
    q_out     receives q (allocated when None; q itself: in place).  q None: only
              k and v are handled, and None is returned.
    q_norm, k_norm [D], of q's type or float32: each head of q (k) is normed before its
              rotation, x / sqrt(mean(x^2) + eps) * weight, in the same pass
    """
    if _lib.elsewhere(k.device):
        with torch.cuda.device(k.device):
            return append_kv_(q, k, v, k_cache, v_cache, slots, positions, cos_sin, q_out, interleaved, q_norm, k_norm, eps)
    if q_norm is not None or k_norm is not None or isinstance(k_cache, QuantizedCache) or isinstance(v_cache, QuantizedCache):
        return _append_rows(q, k, v, k_cache, v_cache, slots, positions, cos_sin, q_out, interleaved, q_norm, k_norm, eps)
    if (torch.is_grad_enabled() and (k.requires_grad or v.requires_grad or k_cache.requires_grad or v_cache.requires_grad
                                     or (q is not None and q.requires_grad)
                                     or (cos_sin is not None and cos_sin.requires_grad))
            or _lib.has_tangent(q, k, v, k_cache, v_cache, cos_sin)):
        raise _lib.no_gradients("append_kv_")
    dev = k.device
    key = (None if q is None else (q.shape, q.stride(), q.dtype, q.device), k.shape, k.stride(), k.dtype, dev, v.shape,
           v.stride(), v.dtype, v.device, k_cache.shape, k_cache.stride(), k_cache.dtype, k_cache.device, v_cache.shape,
           v_cache.stride(), v_cache.dtype, v_cache.device, slots.shape, slots.stride(), slots.dtype, slots.device,
           None if positions is None else (positions.shape, positions.stride(), positions.dtype, positions.device),
           None if cos_sin is None else (cos_sin.shape, cos_sin.stride(), cos_sin.dtype, cos_sin.device),
           None if q_out is None else (q_out.shape, q_out.stride(), q_out.dtype, q_out.device))
    plan = _append_plans.get(key)
    if plan is None:
        plan = _keep(_append_plans, key, _append_plan(q, k, v, k_cache, v_cache, slots, positions, cos_sin, q_out))
    code, T, H, HK, D, R, q_st, k_st, v_st, kc_st, vc_st, o_st, max_pos, pages, page = plan
    if q is not None and q_out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    if T == 0:
        return q_out
    _lib.call("gs_append_kv", code, None if q is None else q.data_ptr(), *q_st, k.data_ptr(), *k_st, v.data_ptr(), *v_st,
              T, H, HK, D, positions.data_ptr() if R else None, cos_sin.data_ptr() if R else None, max_pos, R,
              1 if interleaved else 0, slots.data_ptr(), k_cache.data_ptr(), *kc_st, v_cache.data_ptr(), *vc_st, pages,
              page, None if q is None else q_out.data_ptr(), *o_st, _lib.stream_ptr(dev))
    return q_out


def _append_rows(q, k, v, k_cache, v_cache, slots, positions, cos_sin, q_out, interleaved, q_norm, k_norm,
                 eps) -> torch.Tensor | None:
    """``append_kv_`` with norms of the heads, or into a quantised cache."""
    k_cache, v_cache, k_scales, v_scales = _parts("append_kv_", k_cache, v_cache)
    if (torch.is_grad_enabled() and (k.requires_grad or v.requires_grad or (q is not None and q.requires_grad)
                                     or k_cache.requires_grad or v_cache.requires_grad
                                     or (cos_sin is not None and cos_sin.requires_grad)
                                     or (q_norm is not None and q_norm.requires_grad)
                                     or (k_norm is not None and k_norm.requires_grad))
            or _lib.has_tangent(q, k, v, k_cache, v_cache, cos_sin, q_norm, k_norm)):
        raise _lib.no_gradients("append_kv_")
    interleaved, eps = bool(interleaved), float(eps)       # a tensor's value now, not the tensor
    key = (interleaved, eps, None if q is None else (q.shape, q.stride(), q.dtype, q.device), k.shape, k.stride(), k.dtype,
           k.device, v.shape, v.stride(), v.dtype, v.device, k_cache.shape, k_cache.stride(), k_cache.dtype, k_cache.device,
           v_cache.shape, v_cache.stride(), v_cache.dtype, v_cache.device,
           None if k_scales is None else (k_scales.shape, k_scales.stride(), k_scales.dtype, k_scales.device, v_scales.shape,
                                          v_scales.stride(), v_scales.dtype, v_scales.device),
           slots.shape, slots.stride(), slots.dtype, slots.device,
           None if positions is None else (positions.shape, positions.stride(), positions.dtype, positions.device),
           None if cos_sin is None else (cos_sin.shape, cos_sin.stride(), cos_sin.dtype, cos_sin.device),
           None if q_out is None else (q_out.shape, q_out.stride(), q_out.dtype, q_out.device),
           None if q_norm is None else (q_norm.shape, q_norm.stride(), q_norm.dtype, q_norm.device),
           None if k_norm is None else (k_norm.shape, k_norm.stride(), k_norm.dtype, k_norm.device))
    plan = _rows_plans.get(key)
    if plan is None:
        code, T, H, HK, D, R, q_st, k_st, v_st, kc_st, vc_st, o_st, max_pos, pages, page = _append_plan(
            q, k, v, k_cache, v_cache, slots, positions, cos_sin, q_out, k_scales, v_scales)
        norm_code = _norms_code(q, k, q_norm, k_norm)
        quant = k_scales is not None
        args = _lib.prepared("gs_append_kv_normed", (
            code, None, *q_st, None, *k_st, None, *v_st, T, H, HK, D, None, None, norm_code, eps, None, None, max_pos, R,
            1 if interleaved else 0, None, _lib.GS_DTYPE_E4M3 if quant else code, None, *kc_st, None, *vc_st, None,
            *(k_scales.stride()[:2] if quant else (0, 0)), None, *(v_scales.stride()[:2] if quant else (0, 0)), pages, page,
            None, *o_st, None))
        plan = _keep(_rows_plans, key, (T, R, args))
    T, R, args = plan
    if q is not None and q_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)     # half of torch.empty's time
    if T == 0:
        return q_out
    args = args.copy()                                     # the addresses, where the library's arguments have them
    if q is not None:
        args[1], args[41] = q.data_ptr(), q_out.data_ptr()
        if q_norm is not None:
            args[14] = q_norm.data_ptr()
    args[4], args[7] = k.data_ptr(), v.data_ptr()
    if k_norm is not None:
        args[15] = k_norm.data_ptr()
    if R:
        args[18], args[19] = positions.data_ptr(), cos_sin.data_ptr()
    args[23], args[25], args[29] = slots.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    if k_scales is not None:
        args[33], args[36] = k_scales.data_ptr(), v_scales.data_ptr()
    args[44] = _lib.stream_ptr(k.device)
    _lib.call("gs_append_kv_normed", *args)
    return q_out


def _norms_code(q, k, q_norm, k_norm) -> int:
    """The checks of the norms' weights; their type."""
    who, dtype = "append_kv_", k.dtype
    _on_gpu(who, k.device, q_norm, k_norm)
    if q_norm is not None and q is None:
        raise ValueError(f"{who}: q_norm without q")
    found = None
    for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
        if w is None:
            continue
        if tuple(w.shape) != (k.shape[2],) or not w.is_contiguous() or w.dtype not in (dtype, torch.float32):
            raise ValueError(f"{who}: {name} must be a contiguous tensor [{k.shape[2]}] of {dtype} or float32, got {w.dtype} "
                             f"{tuple(w.shape)}")
        if found is not None and w.dtype != found:
            raise ValueError(f"{who}: q_norm is {found}, k_norm {w.dtype}")
        found = w.dtype
    return _DTYPES[found or dtype]


def _append_plan(q, k, v, k_cache, v_cache, slots, positions, cos_sin, q_out, k_scales=None, v_scales=None) -> tuple:
    """The checks of an ``append_kv_`` call, and its arguments that are not addresses."""
    who = "append_kv_"
    dtype = k.dtype
    if dtype not in _DTYPES:
        raise TypeError(f"{who}: unsupported dtype {dtype}; expected bfloat16 or float32")
    if k.dim() != 3:
        raise ValueError(f"{who}: k must be [tokens, kv_heads, head_dim], got {tuple(k.shape)}")
    T, HK, D = k.shape
    _on_gpu(who, k.device, q, v, k_cache, v_cache, slots, positions, cos_sin, q_out, k_scales, v_scales)
    _heads3(who, "k", k, T, dtype)
    _heads3(who, "v", v, T, dtype)
    if v.shape != k.shape:
        raise ValueError(f"{who}: v is {tuple(v.shape)}, k {tuple(k.shape)}")
    _caches(who, k_cache, v_cache, dtype if k_scales is None else torch.float8_e4m3fn, HK, D)
    if k_scales is not None:
        _scales(who, k_scales, v_scales, k_cache)
    _ints(who, "slots", slots, torch.int64, (T,))
    R = 0
    if cos_sin is not None:
        if cos_sin.dim() != 2 or cos_sin.dtype != torch.float32 or not cos_sin.is_contiguous() or cos_sin.shape[0] == 0:
            raise ValueError(f"{who}: cos_sin must be a contiguous float32 tensor [max_pos, rot_dim], got "
                             f"{cos_sin.dtype} {tuple(cos_sin.shape)}")
        R = cos_sin.shape[1]
        if R % 2 or R > D:
            raise ValueError(f"{who}: cos_sin rotates {R} columns of {D}")
        if positions is None:
            raise ValueError(f"{who}: cos_sin needs positions")
        _ints(who, "positions", positions, torch.int64, (T,))
    H = 0
    if q is not None:
        _heads3(who, "q", q, T, dtype)
        H = q.shape[1]
        if q.shape[2] != D:
            raise ValueError(f"{who}: q has heads of {q.shape[2]}, k of {D}")
        if q_out is not None:
            _heads3(who, "q_out", q_out, T, dtype)
            if q_out.shape != q.shape:
                raise ValueError(f"{who}: q_out is {tuple(q_out.shape)}, q {tuple(q.shape)}")
    elif q_out is not None:
        raise ValueError(f"{who}: q_out without q")
    o_st = (0, 0) if q is None else (H * D, D) if q_out is None else q_out.stride()[:2]
    return (_DTYPES[dtype], T, H, HK, D, R, (0, 0) if q is None else q.stride()[:2], k.stride()[:2], v.stride()[:2],
            k_cache.stride()[:3], v_cache.stride()[:3], o_st, cos_sin.shape[0] if R else 0, k_cache.shape[0],
            k_cache.shape[2])


# ---------------------------------------------------------------------------
# Read
# ---------------------------------------------------------------------------
def read_kv(k_cache, v_cache, slots: torch.Tensor, dtype: torch.dtype | None = None, k_out: torch.Tensor | None = None,
            v_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of the cache by their slots: ``(k, v)`` [T, kv_heads, D], as ``append_kv_`` takes them.

    k_cache, v_cache: tensors, or both ``QuantizedCache``
    slots  [T] int64 (``cache_slots`` with a sequence's whole length gives all its rows);
           one outside the pool gives zeros, and one may come more than once
    dtype  of the result: bfloat16 (the default) or float32 for a quantised cache, whose
           values are exact in both from 2^-126 on; the cache's own otherwise
    k_out, v_out receive the result (allocated when None): views with contiguous head rows
    """
    who = "read_kv"
    if _lib.elsewhere(slots.device):
        with torch.cuda.device(slots.device):
            return read_kv(k_cache, v_cache, slots, dtype, k_out, v_out)
    k_cache, v_cache, k_scales, v_scales = _parts(who, k_cache, v_cache)
    if (torch.is_grad_enabled() and (k_cache.requires_grad or v_cache.requires_grad
                                     or (k_out is not None and k_out.requires_grad)
                                     or (v_out is not None and v_out.requires_grad))
            or _lib.has_tangent(k_cache, v_cache, k_out, v_out)):
        raise _lib.no_gradients(who)
    key = (dtype, k_cache.shape, k_cache.stride(), k_cache.dtype, k_cache.device, v_cache.shape, v_cache.stride(),
           v_cache.dtype, v_cache.device,
           None if k_scales is None else (k_scales.shape, k_scales.stride(), k_scales.dtype, k_scales.device, v_scales.shape,
                                          v_scales.stride(), v_scales.dtype, v_scales.device),
           slots.shape, slots.stride(), slots.dtype, slots.device,
           None if k_out is None else (k_out.shape, k_out.stride(), k_out.dtype, k_out.device),
           None if v_out is None else (v_out.shape, v_out.stride(), v_out.dtype, v_out.device))
    plan = _read_plans.get(key)
    if plan is None:
        plan = _keep(_read_plans, key, _read_plan(k_cache, v_cache, k_scales, v_scales, slots, dtype, k_out, v_out))
    shape, dtype, args = plan
    dev = slots.device
    if k_out is None:
        k_out = slots.new_empty(shape, dtype=dtype)
    if v_out is None:
        v_out = torch.empty_like(k_out, memory_format=torch.contiguous_format)
    if shape[0]:
        args = args.copy()                                 # the addresses, where the library's arguments have them
        args[2], args[6] = k_cache.data_ptr(), v_cache.data_ptr()
        if k_scales is not None:
            args[10], args[13] = k_scales.data_ptr(), v_scales.data_ptr()
        args[20], args[22], args[25], args[28] = slots.data_ptr(), k_out.data_ptr(), v_out.data_ptr(), _lib.stream_ptr(dev)
        _lib.call("gs_read_kv", *args)
    return k_out, v_out


def _read_plan(k_cache, v_cache, k_scales, v_scales, slots, dtype, k_out, v_out) -> tuple:
    """The checks of a ``read_kv`` call, and its arguments that are not addresses."""
    who = "read_kv"
    quant = k_scales is not None
    if dtype is None:
        dtype = torch.bfloat16 if quant else k_cache.dtype
    if dtype not in _DTYPES:
        raise TypeError(f"{who}: unsupported dtype {dtype}; expected bfloat16 or float32")
    if k_cache.dim() != 4 or slots.dim() != 1:
        raise ValueError(f"{who}: a cache is [pages, kv_heads, page_size, head_dim] and slots [tokens], got "
                         f"{tuple(k_cache.shape)} and {tuple(slots.shape)}")
    _on_gpu(who, slots.device, k_cache, v_cache, k_scales, v_scales, k_out, v_out)
    pages, HK, page, D = k_cache.shape
    T = slots.shape[0]
    _caches(who, k_cache, v_cache, torch.float8_e4m3fn if quant else dtype, HK, D)
    if quant:
        _scales(who, k_scales, v_scales, k_cache)
    _ints(who, "slots", slots, torch.int64, (T,))
    for name, t in (("k_out", k_out), ("v_out", v_out)):
        if t is not None:
            _heads3(who, name, t, T, dtype)
            if tuple(t.shape) != (T, HK, D):
                raise ValueError(f"{who}: {name} is {tuple(t.shape)}, expected {(T, HK, D)}")
    code = _DTYPES[dtype]
    return (T, HK, D), dtype, _lib.prepared("gs_read_kv", (
        code, _lib.GS_DTYPE_E4M3 if quant else code, None, *k_cache.stride()[:3], None, *v_cache.stride()[:3], None,
        *(k_scales.stride()[:2] if quant else (0, 0)), None, *(v_scales.stride()[:2] if quant else (0, 0)), pages, page, HK,
        D, None, T, None, *((HK * D, D) if k_out is None else k_out.stride()[:2]), None,
        *((HK * D, D) if v_out is None else v_out.stride()[:2]), None))


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
# One workspace for each stream: calls on one stream follow each other, calls on
# different streams may overlap.  A captured graph may be replayed on any stream,
# beside its capture stream's calls and other graphs: its calls get one of the
# graph's own, from its pool, for each of the capture's streams.  The counters
# start at zero (in a graph: on every replay) and every call leaves them so.
_workspaces: dict = {}
_captured: dict = {}       # by stream: the last capture on it and that capture's buffer


def _new_workspace(device: torch.device, need: int) -> torch.Tensor:
    buf = torch.empty(need, dtype=torch.uint8, device=device)
    buf[:_lib.GS_PAGED_HEAD_BYTES].zero_()     # the rest, up to tens of MB, is written before it is read
    return buf


def _workspace(device: torch.device, stream: int, need: int) -> torch.Tensor:
    key = (device.index, stream)
    if torch.cuda.is_current_stream_capturing():
        capture = _lib.capture_id(stream)
        last, buf = _captured.get(key, (0, None))
        if last != capture or capture == 0 or buf.numel() < need:
            buf = _new_workspace(device, need)
            _captured[key] = (capture, buf)
        return buf
    buf = _workspaces.get(key)
    if buf is None or buf.numel() < need:
        buf = _workspaces[key] = _new_workspace(device, need)
    return buf


_need: dict = {}


def workspace_bytes(dtype: torch.dtype, heads: int, kv_heads: int, head_dim: int, ragged: bool = False) -> int:
    """Workspace of one ``paged_attention`` call (for ``workspace=``), with ``cu_seqlens`` or without; whatever the batch."""
    key = (dtype, heads, kv_heads, head_dim, ragged, torch.cuda.current_device())
    n = _need.get(key)
    if n is None:
        n = int(_lib.load().gs_paged_attention_workspace_bytes(_DTYPES[dtype], heads, kv_heads, head_dim, int(ragged)))
        if n < 0:
            raise _lib.GraniteSwitchError("gs_paged_attention_workspace_bytes", -n, _lib.last_error())
        _need[key] = n
    return n


def paged_attention(q: torch.Tensor, k_cache, v_cache, page_table: torch.Tensor,
                    kv_lens: torch.Tensor, cu_seqlens: torch.Tensor | None = None, scale: float | None = None,
                    window: int = 0, out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                    max_q: int | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the batch's query rows over the paged cache; returns ``out`` [T, heads, D].

    q          [T, heads, D]; heads a multiple of the cache's kv_heads
    k_cache, v_cache: tensors of q's type, or both ``QuantizedCache`` (D a multiple of 16)
    page_table [B, max_pages] int32, kv_lens [B] int32: the sequences' pages and
               lengths, the call's own tokens (already appended) counted
    cu_seqlens [B + 1] int32: sequence s has query rows cu_seqlens[s] ..
               cu_seqlens[s + 1], its last tokens; None: one row per sequence
    scale      of the scores (1 / sqrt(D) when None)
    window     > 0: a row sees the last ``window`` tokens up to its own
    out        receives the result (allocated when None; q itself: in place)
    lse        [T, heads] float32: receives the log of each softmax's total
    max_q      the most query rows of a sequence where the caller knows it: a choice of
               kernels only, one that is too small costs time
    workspace  uint8, ``workspace_bytes`` long, its first 64 KB zeroed before its first
               call, and used by nothing else (one per stream is kept when None)

    A row that sees nothing (an empty sequence), or that is in no sequence (past
    cu_seqlens[B], where a step is padded to a fixed number of rows), gives zeros.
    Keys and values that no row of the call sees may hold anything; a value that is
    not finite may also reach rows of its sequence that come before it.
    """
    dev = q.device
    if _lib.elsewhere(dev):
        with torch.cuda.device(dev):
            return paged_attention(q, k_cache, v_cache, page_table, kv_lens, cu_seqlens, scale, window, out, lse, max_q,
                                   workspace)
    k_cache, v_cache, k_scales, v_scales = _parts("paged_attention", k_cache, v_cache)
    if ((torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad))
            or _lib.has_tangent(q, k_cache, v_cache)):
        raise _lib.no_gradients("paged_attention")
    key = (q.shape, q.stride(), q.dtype, dev, k_cache.shape, k_cache.stride(), k_cache.dtype, k_cache.device,
           v_cache.shape, v_cache.stride(), v_cache.dtype, v_cache.device, page_table.shape, page_table.stride(),
           page_table.dtype, page_table.device, kv_lens.shape, kv_lens.stride(), kv_lens.dtype, kv_lens.device,
           None if cu_seqlens is None else (cu_seqlens.shape, cu_seqlens.stride(), cu_seqlens.dtype, cu_seqlens.device),
           window, max_q, None if out is None else (out.shape, out.stride(), out.dtype, out.device),
           None if lse is None else (lse.shape, lse.stride(), lse.dtype, lse.device),
           None if workspace is None else (workspace.shape, workspace.stride(), workspace.dtype, workspace.device),
           None if k_scales is None else (k_scales.shape, k_scales.stride(), k_scales.dtype, k_scales.device, v_scales.shape,
                                          v_scales.stride(), v_scales.dtype, v_scales.device))
    plan = _attention_plans.get(key)
    if plan is None:
        plan = _keep(_attention_plans, key, _attention_plan(q, k_cache, v_cache, page_table, kv_lens, cu_seqlens, window,
                                                            out, lse, max_q, workspace, k_scales, v_scales))
    code, T, B, H, HK, D, q_st, k_st, v_st, s_st, pages, page, table, o_st, window, most, need, default_scale = plan
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if T == 0:
        return out
    stream = _lib.stream_ptr(dev)
    if workspace is None:
        workspace = _workspace(dev, stream, need)
    scales = () if k_scales is None else (k_scales.data_ptr(), *s_st[:2], v_scales.data_ptr(), *s_st[2:])
    _lib.call("gs_paged_attention_e4m3" if scales else "gs_paged_attention", code, q.data_ptr(), *q_st, k_cache.data_ptr(),
              *k_st, v_cache.data_ptr(), *v_st, *scales, pages, page, page_table.data_ptr(), *table, kv_lens.data_ptr(),
              None if cu_seqlens is None else cu_seqlens.data_ptr(), B, T, most, H, HK, D,
              default_scale if scale is None else scale, window, out.data_ptr(), *o_st,
              None if lse is None else lse.data_ptr(), workspace.data_ptr(), workspace.numel(), stream)
    return out


def check_attended(k_cache, v_cache) -> None:
    """Refuses caches that rows could be stored into but not attended over, by their head dimension or page size."""
    k, _, scales, _ = _parts("paged_attention", k_cache, v_cache)
    page, D = k.shape[2:]
    of = 16 if scales is not None else 8 if k.dtype == torch.bfloat16 else 4
    if D % of or not 0 < D <= 256 or page % 8:
        raise ValueError(f"paged_attention: head_dim={D} must be a multiple of {of} up to 256 and page_size={page} one of 8 "
                         f"(a cache of {'QuantizedCache' if scales is not None else k.dtype})")


def _attention_plan(q, k_cache, v_cache, page_table, kv_lens, cu_seqlens, window, out, lse, max_q, workspace, k_scales,
                    v_scales) -> tuple:
    """The checks of a ``paged_attention`` call, and its arguments that are not addresses."""
    who = "paged_attention"
    dtype = q.dtype
    if dtype not in _DTYPES:
        raise TypeError(f"{who}: unsupported dtype {dtype}; expected bfloat16 or float32")
    _heads3(who, "q", q, None, dtype)
    T, H, D = q.shape
    dev = q.device
    _on_gpu(who, dev, k_cache, v_cache, page_table, kv_lens, cu_seqlens, out, lse, workspace, k_scales, v_scales)
    _caches(who, k_cache, v_cache, dtype if k_scales is None else torch.float8_e4m3fn, None, D)
    if k_scales is not None:
        _scales(who, k_scales, v_scales, k_cache)
    HK = k_cache.shape[1]
    B = kv_lens.shape[0]
    if HK == 0 or H % HK or H == 0:
        raise ValueError(f"{who}: {H} query heads over {HK} key/value heads")
    _ints(who, "kv_lens", kv_lens, torch.int32, (B,))
    _table(who, page_table, B)
    if cu_seqlens is not None:
        _ints(who, "cu_seqlens", cu_seqlens, torch.int32, (B + 1,))
    elif T != B:
        raise ValueError(f"{who}: {T} query rows of {B} sequences without cu_seqlens")
    if window < 0 or (max_q is not None and max_q < 0):
        raise ValueError(f"{who}: window={window} max_q={max_q}")
    if out is not None:
        _heads3(who, "out", out, T, dtype)
        if out.shape != q.shape:
            raise ValueError(f"{who}: out is {tuple(out.shape)}, q {tuple(q.shape)}")
    if lse is not None:
        _ints(who, "lse", lse, torch.float32, (T, H))
    if workspace is not None and (workspace.dtype != torch.uint8 or not workspace.is_contiguous()):
        raise ValueError(f"{who}: workspace must be a contiguous uint8 tensor")
    with torch.cuda.device(dev):
        need = workspace_bytes(dtype, H, HK, D, cu_seqlens is not None) if T else 0
    return (_DTYPES[dtype], T, B, H, HK, D, q.stride()[:2], k_cache.stride()[:3], v_cache.stride()[:3],
            None if k_scales is None else k_scales.stride()[:2] + v_scales.stride()[:2], k_cache.shape[0], k_cache.shape[2],
            (_table_ld(page_table), page_table.shape[1]),
            (H * D, D) if out is None else out.stride()[:2], min(window, _INT32),      # no sequence is longer
            1 if cu_seqlens is None else min(int(max_q or 0), _INT32), need,
            1.0 / math.sqrt(D))


__all__ = ["QuantizedCache", "allocate_cache", "allocate_quantized_cache", "append_kv_", "cache_slots", "check_attended",
           "paged_attention", "read_kv", "rope_table", "workspace_bytes"]
