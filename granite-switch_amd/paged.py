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

Everything is launched on torch's current stream without host synchronisation;
bfloat16 or float32.  No gradients are computed: inputs that autograd tracks are
refused where gradients are enabled.
"""

from __future__ import annotations

import math

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
    return t


def _caches(who: str, k_cache: torch.Tensor, v_cache: torch.Tensor, dtype, kv_heads, head_dim: int):
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        if c.dim() != 4 or c.dtype != dtype or c.shape != k_cache.shape or c.shape[3] != head_dim or \
                (kv_heads is not None and c.shape[1] != kv_heads):
            raise ValueError(f"{who}: {name} must be a {dtype} tensor [pages, kv_heads, page_size, {head_dim}], "
                             f"both caches alike, got {c.dtype} {tuple(c.shape)}")
        if c.stride(3) != 1 and head_dim > 1:
            raise ValueError(f"{who}: {name}'s head dimension must be contiguous (strides {c.stride()})")
    if k_cache.shape[0] == 0 or not 0 < k_cache.shape[2] <= _INT32:
        raise ValueError(f"{who}: pages of {k_cache.shape[2]} rows, {k_cache.shape[0]} of them (1 .. 2^31 - 1 rows)")


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


def append_kv_(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
               slots: torch.Tensor, positions: torch.Tensor | None = None, cos_sin: torch.Tensor | None = None,
               q_out: torch.Tensor | None = None, interleaved: bool = False) -> torch.Tensor | None:
    """Rotate q and k by their positions, store k and v into the cache; returns the rotated q.

    q [T, heads, D], k and v [T, kv_heads, D]: views with contiguous head rows,
    such as slices of the QKV projection's output
    slots     [T] int64: page * page_size + row; one outside the pool (-1) stores
              nothing (padding rows).  No two tokens may share a slot.
    positions [T] int64 and cos_sin [max_pos, R] fp32 (``rope_table``): the first R
              columns of a head are rotated as pairs (j, j + R/2), or (2j, 2j + 1)
              with ``interleaved``, the others copied.  cos_sin None: no rotation.
    q_out     receives q (allocated when None; q itself: in place).  q None: only
              k and v are handled, and None is returned.
    """
    if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad or k_cache.requires_grad or v_cache.requires_grad
                                    or (q is not None and q.requires_grad)
                                    or (cos_sin is not None and cos_sin.requires_grad)):
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


def _append_plan(q, k, v, k_cache, v_cache, slots, positions, cos_sin, q_out) -> tuple:
    """The checks of an ``append_kv_`` call, and its arguments that are not addresses."""
    who = "append_kv_"
    dtype = k.dtype
    if dtype not in _DTYPES:
        raise TypeError(f"{who}: unsupported dtype {dtype}; expected bfloat16 or float32")
    if k.dim() != 3:
        raise ValueError(f"{who}: k must be [tokens, kv_heads, head_dim], got {tuple(k.shape)}")
    T, HK, D = k.shape
    _on_gpu(who, k.device, q, v, k_cache, v_cache, slots, positions, cos_sin, q_out)
    _heads3(who, "k", k, T, dtype)
    _heads3(who, "v", v, T, dtype)
    if v.shape != k.shape:
        raise ValueError(f"{who}: v is {tuple(v.shape)}, k {tuple(k.shape)}")
    _caches(who, k_cache, v_cache, dtype, HK, D)
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


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    kv_lens: torch.Tensor, cu_seqlens: torch.Tensor | None = None, scale: float | None = None,
                    window: int = 0, out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                    max_q: int | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the batch's query rows over the paged cache; returns ``out`` [T, heads, D].

    q          [T, heads, D]; heads a multiple of the cache's kv_heads
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
    if torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad):
        raise _lib.no_gradients("paged_attention")
    dev = q.device
    key = (q.shape, q.stride(), q.dtype, dev, k_cache.shape, k_cache.stride(), k_cache.dtype, k_cache.device,
           v_cache.shape, v_cache.stride(), v_cache.dtype, v_cache.device, page_table.shape, page_table.stride(),
           page_table.dtype, page_table.device, kv_lens.shape, kv_lens.stride(), kv_lens.dtype, kv_lens.device,
           None if cu_seqlens is None else (cu_seqlens.shape, cu_seqlens.stride(), cu_seqlens.dtype, cu_seqlens.device),
           window, max_q, None if out is None else (out.shape, out.stride(), out.dtype, out.device),
           None if lse is None else (lse.shape, lse.stride(), lse.dtype, lse.device),
           None if workspace is None else (workspace.shape, workspace.stride(), workspace.dtype, workspace.device))
    plan = _attention_plans.get(key)
    if plan is None:
        plan = _keep(_attention_plans, key, _attention_plan(q, k_cache, v_cache, page_table, kv_lens, cu_seqlens, window,
                                                            out, lse, max_q, workspace))
    code, T, B, H, HK, D, q_st, k_st, v_st, pages, page, table, o_st, window, most, need, default_scale = plan
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    if T == 0:
        return out
    stream = _lib.stream_ptr(dev)
    if workspace is None:
        workspace = _workspace(dev, stream, need)
    _lib.call("gs_paged_attention", code, q.data_ptr(), *q_st, k_cache.data_ptr(), *k_st, v_cache.data_ptr(), *v_st, pages,
              page, page_table.data_ptr(), *table, kv_lens.data_ptr(), None if cu_seqlens is None else cu_seqlens.data_ptr(),
              B, T, most, H, HK, D, default_scale if scale is None else scale, window, out.data_ptr(), *o_st,
              None if lse is None else lse.data_ptr(), workspace.data_ptr(), workspace.numel(), stream)
    return out


def _attention_plan(q, k_cache, v_cache, page_table, kv_lens, cu_seqlens, window, out, lse, max_q, workspace) -> tuple:
    """The checks of a ``paged_attention`` call, and its arguments that are not addresses."""
    who = "paged_attention"
    dtype = q.dtype
    if dtype not in _DTYPES:
        raise TypeError(f"{who}: unsupported dtype {dtype}; expected bfloat16 or float32")
    _heads3(who, "q", q, None, dtype)
    T, H, D = q.shape
    dev = q.device
    _on_gpu(who, dev, k_cache, v_cache, page_table, kv_lens, cu_seqlens, out, lse, workspace)
    _caches(who, k_cache, v_cache, dtype, None, D)
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
    return (_DTYPES[dtype], T, B, H, HK, D, q.stride()[:2], k_cache.stride()[:3], v_cache.stride()[:3], k_cache.shape[0],
            k_cache.shape[2], (_table_ld(page_table), page_table.shape[1]),
            (H * D, D) if out is None else out.stride()[:2], min(window, _INT32),      # no sequence is longer
            1 if cu_seqlens is None else min(int(max_q or 0), _INT32), need,
            1.0 / math.sqrt(D))


__all__ = ["allocate_cache", "append_kv_", "cache_slots", "paged_attention", "rope_table", "workspace_bytes"]
