"""The residual add between two blocks of a decoder layer with the norms around it, in one pass.

    b  = x                                     the block's output
    b  = rms(b) * post_weight                  norm after the block (optional)
    b  = b * act(gate)                         gate (optional)
    r' = residual + scale * b                  residual stream, scaled
    y  = rms(r') * weight                      norm before the next block

with rms(t) = t * rsqrt(mean(t^2) + eps).  Sums and r' are held in fp32; y is
taken from r' before r' is rounded.  Launched on torch's current stream without
host synchronisation.  No gradients are computed: inputs that autograd tracks are
refused where gradients are enabled.
"""

from __future__ import annotations

import math

import torch

from . import _lib

_DTYPES = {torch.bfloat16: _lib.GS_DTYPE_BF16, torch.float32: _lib.GS_DTYPE_FP32}
_ACTS = {None: _lib.GS_GATE_NONE, "sigmoid": _lib.GS_GATE_SIGMOID, "tanh": _lib.GS_GATE_TANH}


# What a call's checks found, by the shapes, strides, types and devices of its
# tensors (never by their addresses): a serving loop's calls repeat a few, and the
# checks take longer than a small call's kernel.
_plans: dict = {}
_PLAN_CAP = 4096


def _rows(name: str, t: torch.Tensor, shape, dtype) -> torch.Tensor:
    if t.shape != shape or t.dtype not in (dtype if isinstance(dtype, tuple) else (dtype,)):
        raise ValueError(f"residual_norm: {name} is {t.dtype} {tuple(t.shape)}, expected {dtype} {tuple(shape)}")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"residual_norm: {name} rows must be contiguous (strides {t.stride()})")
    return t


def _ld(t: torch.Tensor) -> int:
    """Row stride of a matrix (a single row's stride says nothing)."""
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def residual_norm(x: torch.Tensor | None, residual: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5,
                  scale: float = 1.0, gate: torch.Tensor | None = None, post_weight: torch.Tensor | None = None,
                  gate_act: str | None = None, out: torch.Tensor | None = None,
                  residual_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(y, r')`` of a block's output ``x`` and the residual stream.

    x:        [..., hidden] bfloat16 or float32; None: y is the norm of the
              residual alone, and the residual is returned as it is
    residual: as x, or float32 (a residual stream held in 32 bits)
    weight, post_weight: [hidden], x's dtype or float32 (both the same)
    gate:     broadcastable to x: [hidden], [..., 1] or [..., hidden], x's dtype;
              ``gate_act`` None, "sigmoid" or "tanh" is applied to it
    out, residual_out: results (allocated when None); ``residual_out=residual``
              updates the stream in place, ``out=x`` reuses x
    """
    if torch.is_grad_enabled() and (residual.requires_grad or weight.requires_grad
                                    or (x is not None and x.requires_grad) or (gate is not None and gate.requires_grad)
                                    or (post_weight is not None and post_weight.requires_grad)):
        raise _lib.no_gradients("residual_norm")
    if x is not None and x.dim() == 2 and residual.dim() == 2:
        key = (x.shape, x.stride(), x.dtype, x.device, residual.shape, residual.stride(), residual.dtype, residual.device,
               weight.shape, weight.stride(), weight.dtype, weight.device,
               None if gate is None else (gate.shape, gate.stride(), gate.dtype, gate.device), gate_act,
               None if post_weight is None else (post_weight.shape, post_weight.stride(), post_weight.dtype, post_weight.device),
               None if out is None else (out.shape, out.stride(), out.dtype, out.device),
               None if residual_out is None else (residual_out.shape, residual_out.stride(), residual_out.dtype,
                                                  residual_out.device))
        plan = _plans.get(key)
        if plan is not None:
            code, r_code, w_code, act, g_st, ldx, ldr, ldro, ldy, rows, hidden = plan
            dev = x.device
            y = torch.empty(x.shape, dtype=x.dtype, device=dev) if out is None else out
            r = torch.empty(x.shape, dtype=residual.dtype, device=dev) if residual_out is None else residual_out
            if rows and hidden:
                _lib.call("gs_residual_norm", code, x.data_ptr(), ldx, residual.data_ptr(), ldr, r_code,
                          None if gate is None else gate.data_ptr(), *g_st, act,
                          None if post_weight is None else post_weight.data_ptr(), weight.data_ptr(), w_code, eps, scale,
                          rows, hidden, r.data_ptr(), ldro, y.data_ptr(), ldy, _lib.stream_ptr(dev))
            return y, r
    else:
        key = None
    act = _ACTS.get(gate_act, -1) if gate_act is None or isinstance(gate_act, str) else -1
    if act < 0:
        raise ValueError(f"residual_norm: gate_act={gate_act!r} (None, 'sigmoid' or 'tanh')")
    like = residual if x is None else x
    if not like.is_cuda or not residual.is_cuda:
        raise ValueError("residual_norm: tensors must live on the GPU")
    if x is None and (gate is not None or post_weight is not None):
        raise ValueError("residual_norm: gate and post_weight need x")
    if x is not None and x.shape != residual.shape:
        raise ValueError(f"residual_norm: x {tuple(x.shape)} and residual {tuple(residual.shape)} differ")
    if residual.dim() == 0:
        raise ValueError("residual_norm: residual must have a hidden dimension")
    hidden = residual.shape[-1]
    if hidden >= 2 ** 31:
        raise ValueError(f"residual_norm: hidden={hidden} (up to 2^31 - 1)")
    if weight.dtype in _DTYPES and x is None and out is not None:
        dtype = out.dtype
    else:
        dtype = like.dtype
    if dtype not in _DTYPES:
        raise TypeError(f"residual_norm: unsupported dtype {dtype}; expected bfloat16 or float32")
    if residual.dtype not in (dtype, torch.float32):
        raise TypeError(f"residual_norm: residual is {residual.dtype} beside {dtype}")
    for name, w in (("weight", weight), ("post_weight", post_weight)):
        if w is None:
            continue
        if w.shape != (hidden,) or not w.is_contiguous() or w.dtype not in (dtype, torch.float32) or w.dtype != weight.dtype:
            raise ValueError(f"residual_norm: {name} must be a contiguous [{hidden}] tensor of {dtype} or float32, both "
                             f"weights alike, got {w.dtype} {tuple(w.shape)}")
    shape = residual.shape
    rows = math.prod(shape[:-1])
    for t in (x, weight, gate, post_weight, out, residual_out):
        if t is not None and t.device != residual.device:
            raise ValueError("residual_norm: tensors must live on one GPU")

    def flat(t):
        return t if t.dim() == 2 else t.reshape(rows, hidden)

    def flat_out(name, t, dt):
        if t is None:
            return None
        if t.shape != shape or t.dtype != dt:
            raise ValueError(f"residual_norm: {name} is {t.dtype} {tuple(t.shape)}, expected {dt} {tuple(shape)}")
        return t if t.dim() == 2 else t.view(rows, hidden)      # raises where a copy would be needed

    r2 = flat(residual)
    _rows("residual", r2, r2.shape, residual.dtype)
    x2 = None if x is None else _rows("x", flat(x), r2.shape, dtype)
    y2 = flat_out("out", out, dtype)
    if y2 is None:
        y2 = torch.empty(rows, hidden, dtype=dtype, device=residual.device)
    else:
        _rows("out", y2, r2.shape, dtype)
    ro2 = None
    if x is not None:
        ro2 = flat_out("residual_out", residual_out, residual.dtype)
        if ro2 is None:
            ro2 = torch.empty(rows, hidden, dtype=residual.dtype, device=residual.device)
        else:
            _rows("residual_out", ro2, r2.shape, residual.dtype)
    g_row = g_col = 0
    given_gate = gate
    if gate is not None:
        if gate.dtype != dtype:
            raise TypeError(f"residual_norm: gate is {gate.dtype}, expected {dtype}")
        g = gate.expand(shape)
        if g.dim() != 2:
            g = gate.reshape(1, -1).expand(rows, hidden) if gate.numel() == hidden and gate.shape[-1] == hidden \
                else gate.expand(*shape[:-1], gate.shape[-1]).reshape(rows, gate.shape[-1]).expand(rows, hidden)
        g_row, g_col = (g.stride(0) if rows > 1 else 0), (g.stride(1) if hidden > 1 else 0)
        if g_col not in (0, 1):
            g = g.contiguous()
            g_row, g_col = hidden, 1
        gate = g
    if key is not None and (gate is None or gate.data_ptr() == given_gate.data_ptr()):
        if len(_plans) >= _PLAN_CAP:
            _plans.clear()
        _plans[key] = (_DTYPES[dtype], _DTYPES[residual.dtype], _DTYPES[weight.dtype], act, (g_row, g_col), _ld(x2), _ld(r2),
                       _ld(ro2), _ld(y2), rows, hidden)
    if rows and hidden:
        _lib.call("gs_residual_norm", _DTYPES[dtype], _lib.ptr(x2), 0 if x2 is None else _ld(x2), r2.data_ptr(), _ld(r2),
                  _DTYPES[residual.dtype], _lib.ptr(gate), g_row, g_col, act, _lib.ptr(post_weight), weight.data_ptr(),
                  _DTYPES[weight.dtype], float(eps), float(scale), rows, hidden, _lib.ptr(ro2),
                  0 if ro2 is None else _ld(ro2), y2.data_ptr(), _ld(y2), _lib.stream_ptr(residual.device))
    y = out if out is not None else (y2 if residual.dim() == 2 else y2.view(shape))
    if x is None:
        return y, residual
    return y, residual_out if residual_out is not None else (ro2 if residual.dim() == 2 else ro2.view(shape))


