"""ctypes binding of libgranite_switch_amd.so (the C ABI in include/granite_switch_amd.h).

The library is loaded after torch, so it binds to the HIP runtime torch
already mapped (same soname) and every launch can go on torch's current
stream.  There is no fallback: if the library is missing, every entry point
raises.
"""

from __future__ import annotations

import ctypes
import os
import threading

import torch  # must be imported before the HIP library is loaded
from torch.autograd import forward_ad

from .build import LIB_PATH

c_void_p = ctypes.c_void_p
c_i32 = ctypes.c_int32
c_i64 = ctypes.c_int64

GS_OK = 0
GS_ERR_INVALID = 1
GS_ERR_HIP = 2
GS_ERR_WORKSPACE = 3
GS_DTYPE_BF16 = 0
GS_DTYPE_FP32 = 1
GS_DTYPE_E4M3 = 2
GS_MAX_ADAPTERS = 256
GS_MAX_SLICES = 8
GS_MAX_RANK = 512
GS_RANK_CLASS_SPLIT = 64
GS_NOALLOC_SCRATCH_BYTES = 64 << 20
GS_PAGED_HEAD_BYTES = 65536
GS_GATE_NONE = 0
GS_GATE_SIGMOID = 1
GS_GATE_TANH = 2

# name -> (restype, argtypes); mirrors include/granite_switch_amd.h
SIGNATURES = {
    "gs_version": (c_i32, []),
    "gs_last_error": (ctypes.c_char_p, []),
    "gs_build_segments_workspace_bytes": (c_i64, [c_i64, c_i32]),
    "gs_build_segments": (c_i32, [c_void_p, c_void_p, c_void_p, c_void_p, c_i64, c_i32, c_i32, c_void_p, c_void_p,
                                  c_void_p, c_void_p, c_i64, c_void_p]),
    "gs_route_latest_wins": (c_i32, [c_void_p, c_void_p, c_i64, c_i32, c_void_p, c_i32, c_i32, c_void_p, c_void_p,
                                     c_void_p]),
    "gs_shrink_workspace_bytes": (c_i64, [c_i64, c_i32, c_i32, c_i32, c_i32, c_void_p]),
    "gs_shrink_ksplits": (c_i32, [c_i32, c_i64, c_i32, c_i32, c_i32, c_i32, c_void_p, c_void_p]),
    "gs_switched_lora_pair": (c_i32, [c_i32, c_i64, c_i32, c_i32, c_void_p, c_i32, c_i32, c_i32, c_void_p]),
    "gs_expand_span_tiles": (c_i32, [c_i64, c_i32, c_i32, c_i32, c_void_p]),
    "gs_check_segment_addresses": (c_i64, [c_i32, c_i64, c_i32, c_i64, c_i32, c_i64, c_void_p, c_i32, c_void_p, c_i64,
                                           c_void_p, c_i64, c_void_p, c_i32, c_i32, c_void_p, c_void_p, c_void_p,
                                           c_i64, ctypes.c_char_p, c_i64, c_void_p]),
    "gs_check_gemm_addresses": (c_i64, [c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, ctypes.c_char_p, c_i64, c_void_p]),
    "gs_check_token_addresses": (c_i64, [c_i64, c_i32, c_void_p, c_i32, c_void_p, c_i32, c_i32, c_i32, c_i32,
                                         ctypes.c_char_p, c_i64, c_void_p]),
    "gs_check_build_addresses": (c_i64, [c_i64, c_i32, c_i32, c_void_p, c_void_p, c_void_p, c_void_p, c_i32,
                                         ctypes.c_char_p, c_i64, c_void_p]),
    "gs_check_small_addresses": (c_i64, [c_i32, c_i64, c_i32, c_i64, c_i32, c_i64, c_void_p, c_i32, c_void_p, c_i64,
                                         c_void_p, c_i64, c_void_p, c_i32, c_i32, c_void_p, c_i32, c_i32, c_i32,
                                         ctypes.c_char_p, c_i64, c_void_p]),
    "gs_check_xext_addresses": (c_i64, [c_i32, c_i64, c_i64, c_i64, c_void_p, c_i32, c_void_p, c_i64, c_i64, c_i64,
                                        c_void_p, c_i64, c_void_p, c_void_p, c_i32, c_i32, c_i32, c_i32, c_i64, c_i32,
                                        ctypes.c_char_p, c_i64, c_void_p]),
    "gs_shrink": (c_i32, [c_i32, c_void_p, c_i64, c_i64, c_i32, c_void_p, c_void_p, c_void_p, c_i32, c_i32, c_i32,
                          c_void_p, c_void_p, c_void_p, c_void_p, c_i64, c_void_p, c_i64, c_void_p]),
    "gs_expand_add": (c_i32, [c_i32, c_void_p, c_i64, c_i64, c_i32, c_void_p, c_i32, c_void_p, c_i64, c_i32, c_void_p,
                              c_void_p, c_void_p, c_void_p, c_i32, c_i32, c_void_p, c_void_p, c_void_p, c_void_p]),
    "gs_switched_lora": (c_i32, [c_i32, c_void_p, c_i64, c_void_p, c_i64, c_i64, c_i32, c_i32, c_void_p, c_i32,
                                 c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_i32, c_i32, c_void_p, c_void_p,
                                 c_void_p, c_void_p, c_void_p, c_i64, c_void_p]),
    "gs_switched_lora_noalloc": (c_i32, [c_i32, c_void_p, c_i64, c_void_p, c_i64, c_i64, c_i32, c_i32, c_void_p,
                                         c_i32, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_i32, c_i32,
                                         c_void_p, c_void_p, c_void_p, c_void_p]),
    "gs_small_eligible": (c_i32, [c_i64, c_i32, c_i32, c_void_p, c_i32, c_i32]),
    "gs_small_workspace_bytes": (c_i64, [c_i32, c_i64, c_i32, c_i32, c_i32, c_i32, c_i32, c_void_p]),
    "gs_small_sync_bytes": (c_i64, []),
    "gs_small_set_wait_limit": (c_i64, [c_i64]),
    "gs_small_workgroups": (c_i64, [c_i32, c_i64, c_i32, c_i32, c_i32, c_i32, c_i32, c_void_p, c_i32]),
    "gs_switched_lora_small": (c_i32, [c_i32, c_void_p, c_void_p, c_void_p, c_void_p, c_i32, c_void_p, c_void_p,
                                       c_i64, c_void_p, c_i64, c_i64, c_i32, c_i32, c_void_p, c_i32, c_void_p,
                                       c_void_p, c_void_p, c_void_p, c_void_p, c_i32, c_i32, c_void_p, c_i64,
                                       c_void_p, c_i64, c_i32, c_i32, c_void_p]),
    "gs_compute_bitmasks": (c_i32, [c_void_p, c_i32, c_i64, c_void_p, c_i32, c_i32, c_i32, c_void_p, c_void_p,
                                    c_void_p]),
    "gs_bitmask_table_form": (c_i32, [c_i64, c_i32, c_i32, c_i32]),
    "gs_switch_lora_expand": (c_i32, [c_void_p, c_i64, c_i64, c_i64, c_void_p, c_i32, c_void_p, c_i64, c_void_p,
                                      c_void_p, c_void_p, c_void_p, c_i32, c_i32, c_i32, c_void_p]),
    "gs_switch_lora_expand_swiglu": (c_i32, [c_void_p, c_i64, c_i64, c_void_p, c_i64, c_i64, c_i64, c_void_p, c_i32,
                                             c_void_p, c_i64, c_void_p, c_void_p, c_void_p, c_i32, c_i32, c_i32, c_i32,
                                             c_void_p]),
    "gs_split_adapter_indices": (c_i32, [c_void_p, c_i32, c_void_p, c_i32, c_i64, c_void_p, c_void_p, c_void_p]),
    "gs_switch_lora_shrink_expand": (c_i32, [c_void_p, c_i32, c_i64, c_i64, c_void_p, c_i64, c_i64, c_i64, c_void_p,
                                             c_i32, c_void_p, c_i64, c_void_p, c_void_p, c_void_p, c_void_p, c_i32,
                                             c_i32, c_i32, c_void_p]),
    "gs_gemm_bf16_tn": (c_i32, [c_void_p, c_i64, c_void_p, c_i64, c_void_p, c_i64, c_i64, c_i64, c_i64, c_void_p]),
    "gs_append_kv": (c_i32, [c_i32] + [c_void_p, c_i64, c_i64] * 3 + [c_i64, c_i32, c_i32, c_i32, c_void_p, c_void_p,
                             c_i64, c_i32, c_i32, c_void_p] + [c_void_p, c_i64, c_i64, c_i64] * 2
                     + [c_i64, c_i32, c_void_p, c_i64, c_i64, c_void_p]),
    "gs_append_kv_normed": (c_i32, [c_i32] + [c_void_p, c_i64, c_i64] * 3 + [c_i64, c_i32, c_i32, c_i32, c_void_p, c_void_p,
                                    c_i32, ctypes.c_float, c_void_p, c_void_p, c_i64, c_i32, c_i32, c_void_p, c_i32]
                            + [c_void_p, c_i64, c_i64, c_i64] * 2 + [c_void_p, c_i64, c_i64] * 2
                            + [c_i64, c_i32, c_void_p, c_i64, c_i64, c_void_p]),
    "gs_read_kv": (c_i32, [c_i32, c_i32] + [c_void_p, c_i64, c_i64, c_i64] * 2 + [c_void_p, c_i64, c_i64] * 2
                   + [c_i64, c_i32, c_i32, c_i32, c_void_p, c_i64] + [c_void_p, c_i64, c_i64] * 2 + [c_void_p]),
    "gs_cache_slots": (c_i32, [c_void_p, c_i64, c_i32, c_i64, c_i32, c_void_p, c_void_p, c_i32, c_i64, c_void_p,
                               c_void_p, c_void_p]),
    "gs_paged_attention_workspace_bytes": (c_i64, [c_i32, c_i32, c_i32, c_i32, c_i32]),
    "gs_paged_attention": (c_i32, [c_i32, c_void_p, c_i64, c_i64] + [c_void_p, c_i64, c_i64, c_i64] * 2
                           + [c_i64, c_i32, c_void_p, c_i64, c_i32, c_void_p, c_void_p, c_i32, c_i64, c_i32, c_i32,
                              c_i32, c_i32, ctypes.c_float, c_i32, c_void_p, c_i64, c_i64, c_void_p, c_void_p, c_i64,
                              c_void_p]),
    "gs_paged_attention_e4m3": (c_i32, [c_i32, c_void_p, c_i64, c_i64] + [c_void_p, c_i64, c_i64, c_i64] * 2
                                + [c_void_p, c_i64, c_i64] * 2
                                + [c_i64, c_i32, c_void_p, c_i64, c_i32, c_void_p, c_void_p, c_i32, c_i64, c_i32, c_i32,
                                   c_i32, c_i32, ctypes.c_float, c_i32, c_void_p, c_i64, c_i64, c_void_p, c_void_p, c_i64,
                                   c_void_p]),
    "gs_capture_id": (c_i32, [c_void_p, c_void_p]),
    "gs_check_paged_addresses": (c_i64, [c_i32] + [c_i64] * 9 + [c_i32, c_void_p, c_i64, c_i32, c_void_p, c_void_p,
                                         c_i32, c_i64, c_i32, c_i32, c_i32, c_i32, c_i64, c_i64, c_i32,
                                         ctypes.c_char_p, c_i64, c_void_p]),
    "gs_check_append_addresses": (c_i64, [c_i32, c_i32] + [c_i64] * 5 + [c_i32, c_i32, c_i32, c_void_p, c_i64, c_i32,
                                          c_i32, c_void_p] + [c_i64] * 4 + [c_i32, c_i32, ctypes.c_char_p, c_i64,
                                          c_void_p]),
    "gs_check_paged_e4m3_addresses": (c_i64, [c_i32] + [c_i64] * 11 + [c_i32, c_void_p, c_i64, c_i32, c_void_p, c_void_p,
                                              c_i32, c_i64, c_i32, c_i32, c_i32, c_i32, c_i64, c_i64, c_i32,
                                              ctypes.c_char_p, c_i64, c_void_p]),
    "gs_check_rows_addresses": (c_i64, [c_i32, c_i32, c_i32] + [c_i64] * 5 + [c_i32, c_i32, c_i32, c_void_p, c_i64, c_i32,
                                        c_i32, c_void_p] + [c_i64] * 6 + [c_i32, c_i32, ctypes.c_char_p, c_i64, c_void_p]),
    "gs_residual_norm": (c_i32, [c_i32, c_void_p, c_i64, c_void_p, c_i64, c_i32, c_void_p, c_i64, c_i64, c_i32,
                                 c_void_p, c_void_p, c_i32, ctypes.c_float, ctypes.c_float, c_i64, c_i32, c_void_p,
                                 c_i64, c_void_p, c_i64, c_void_p]),
    "gs_gemm_form": (c_i32, [c_i64, c_i64, c_i64, c_i64, c_i64, c_i32, c_void_p]),
}


class GraniteSwitchError(RuntimeError):
    """A library entry point returned a non-OK status."""

    def __init__(self, func: str, status: int, message: str):
        super().__init__(f"{func} failed (status {status}): {message}")
        self.func = func
        self.status = status


_lock = threading.Lock()
_lib = None


def load() -> ctypes.CDLL:
    """Load (once) and return the library; raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        if not os.path.exists(LIB_PATH):
            raise ImportError(
                f"{LIB_PATH} is missing: build it with __graft_entry__.build() or "
                "python granite-switch_amd/build.py (there is no CPU fallback)")
        lib = ctypes.CDLL(LIB_PATH, mode=ctypes.RTLD_LOCAL)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib


def last_error() -> str:
    msg = load().gs_last_error()
    return msg.decode() if msg else ""


def call(name: str, *args) -> int:
    """Call an entry point; raise GraniteSwitchError on a non-OK status."""
    lib = load()
    rc = getattr(lib, name)(*args)
    if rc != GS_OK:
        msg = lib.gs_last_error()
        raise GraniteSwitchError(name, rc, msg.decode() if msg else "")
    return rc


def prepared(name: str, args) -> list:
    """A call's arguments as the binding has them: those that repeat are converted once (a third of a long call's time)."""
    return [a if a is None or t is c_void_p else t(a) for a, t in zip(args, SIGNATURES[name][1], strict=True)]


# the stream's handle without a Stream object around it (a launch asks once)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_ptr(device: torch.device | None = None) -> int:
    """hipStream_t of torch's current stream on ``device``."""
    if device is not None and device.index is not None and _raw_stream is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def elsewhere(dev: torch.device) -> bool:
    """Whether ``dev`` is a GPU that is not the current one: a launch goes to the current one's queues."""
    return dev.type == "cuda" and dev.index is not None and dev.index != torch.cuda.current_device()


def capture_id(stream: int) -> int:
    """The id of the graph capture that ``stream`` is part of; 0: none."""
    found = c_i64()
    call("gs_capture_id", stream, ctypes.byref(found))
    return found.value


def no_gradients(who: str) -> RuntimeError:
    """For a call whose inputs autograd tracks: their gradients would be lost silently."""
    return RuntimeError(f"{who} computes no gradients: call it under torch.no_grad() / torch.inference_mode(), or with "
                        "tensors that do not require grad and have no forward-mode tangent")


def has_tangent(*ts) -> bool:
    """Whether one of the tensors (or None) is a dual one of forward-mode differentiation: ``requires_grad`` says nothing
    of its tangent, and ``no_grad`` does not end it."""
    if forward_ad._current_level < 0:
        return False
    # a registered op's body runs below autograd, where no tangent can be asked for: look from above it
    with torch._C._ForceDispatchKeyGuard(torch._C._dispatch_tls_local_include_set(),
                                         torch._C.DispatchKeySet(torch._C.DispatchKey.Undefined)):
        return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts)


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()
