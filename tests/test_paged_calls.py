"""CPU tests: what the entry points of the paged cache and the norms refuse, and their ops' shapes.

No kernel is launched: every library call here is rejected by its argument
checks before any HIP call, or has no rows.
"""

from __future__ import annotations

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from granite_switch_amd import _lib, decoder, norms, ops, paged, vllm_layers

P = ctypes.c_void_p(4096)                                  # an address that no check reads from
BF16, FP32 = _lib.GS_DTYPE_BF16, _lib.GS_DTYPE_FP32

ATTENTION = dict(dtype=BF16, q=P, q_ts=1024, q_hs=128, k=P, k_ps=16384, k_hs=2048, k_rs=128, v=P, v_ps=16384, v_hs=2048,
                 v_rs=128, num_pages=4, page_size=16, table=P, ld_table=4, max_pages=4, lens=P, cu=None, num_seqs=2,
                 num_tokens=2, max_q=1, heads=8, kv_heads=2, head_dim=128, scale=1.0, window=0, out=P, o_ts=1024,
                 o_hs=128, lse=None, ws=P, ws_bytes=1 << 40, stream=None)
APPEND = dict(dtype=BF16, q=P, q_ts=1024, q_hs=128, k=P, k_ts=256, k_hs=128, v=P, v_ts=256, v_hs=128, num_tokens=2,
              heads=8, kv_heads=2, head_dim=128, positions=P, cos_sin=P, max_pos=64, rot_dim=128, interleaved=0, slots=P,
              k_cache=P, kc_ps=4096, kc_hs=2048, kc_rs=128, v_cache=P, vc_ps=4096, vc_hs=2048, vc_rs=128, num_pages=4,
              page_size=16, q_out=P, o_ts=1024, o_hs=128, stream=None)
NORM = dict(dtype=BF16, x=P, ldx=256, residual=ctypes.c_void_p(1 << 20), ldr=256, residual_dtype=BF16, gate=None,
            gate_row=0, gate_col=0, gate_act=_lib.GS_GATE_NONE, post_weight=None, weight=ctypes.c_void_p(2 << 20),
            weight_dtype=BF16, eps=1e-5, scale=1.0, rows=2, hidden=256, residual_out=ctypes.c_void_p(3 << 20), ldro=256,
            y=ctypes.c_void_p(4 << 20), ldy=256, stream=None)
SLOTS = dict(table=P, ld_table=4, max_pages=4, num_pages=4, page_size=16, lens=P, cu=None, num_seqs=2, num_tokens=2,
             slots=P, positions=P, stream=None)


def _refused(name, base, change):
    unknown = set(change) - set(base)
    assert not unknown, unknown
    with pytest.raises(_lib.GraniteSwitchError) as e:
        _lib.call(name, *{**base, **change}.values())
    return e.value


@pytest.mark.parametrize("change", [
    dict(dtype=7), dict(num_tokens=-1), dict(num_tokens=3), dict(heads=7), dict(kv_heads=0), dict(head_dim=264),
    dict(head_dim=100), dict(page_size=12), dict(num_pages=0), dict(ld_table=3), dict(window=-1), dict(max_q=-1),
    dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(lens=None), dict(table=None),
    dict(q=ctypes.c_void_p(4104)), dict(k_rs=129), dict(o_ts=1028), dict(q_hs=-128)], ids=str)
def test_attention_arguments(change):
    e = _refused("gs_paged_attention", ATTENTION, change)
    assert e.status == _lib.GS_ERR_INVALID and "gs_paged_attention" in str(e)


@pytest.mark.parametrize("sizes", [(7, 8, 2, 128), (BF16, 7, 2, 128), (BF16, 8, 0, 128), (FP32, 8, 2, 257), (FP32, 8, 2, 0)])
def test_workspace_arguments(sizes):
    lib = _lib.load()
    assert lib.gs_paged_attention_workspace_bytes(*sizes, 0) == -_lib.GS_ERR_INVALID
    assert "gs_paged_attention_workspace_bytes" in _lib.last_error()


@pytest.mark.parametrize("change", [
    dict(dtype=7), dict(num_tokens=-1), dict(kv_heads=0), dict(head_dim=513), dict(rot_dim=130), dict(rot_dim=63),
    dict(page_size=0), dict(num_pages=0), dict(k=None), dict(v=None), dict(slots=None), dict(k_cache=None),
    dict(v_cache=None), dict(q_out=None), dict(positions=None), dict(cos_sin=None), dict(max_pos=0)], ids=str)
def test_append_arguments(change):
    e = _refused("gs_append_kv", APPEND, change)
    assert e.status == _lib.GS_ERR_INVALID and "gs_append_kv" in str(e)


@pytest.mark.parametrize("change", [dict(num_tokens=-1), dict(num_seqs=-1), dict(page_size=0), dict(ld_table=3),
                                    dict(slots=None), dict(positions=None), dict(lens=None)], ids=str)
def test_slots_arguments(change):
    e = _refused("gs_cache_slots", SLOTS, change)
    assert e.status == _lib.GS_ERR_INVALID and "gs_cache_slots" in str(e)


@pytest.mark.parametrize("change", [
    dict(dtype=7), dict(residual_dtype=5), dict(dtype=FP32, weight_dtype=BF16, residual_dtype=FP32), dict(rows=-1),
    dict(hidden=0), dict(gate_act=9), dict(eps=-1.0), dict(residual=None), dict(weight=None), dict(y=None),
    dict(residual_out=None), dict(ldx=255), dict(ldy=255), dict(x=None, gate=P), dict(gate=P, gate_col=2),
    dict(y=ctypes.c_void_p((3 << 20) + 64))], ids=str)
def test_norm_arguments(change):
    e = _refused("gs_residual_norm", NORM, change)
    assert e.status == _lib.GS_ERR_INVALID and "gs_residual_norm" in str(e)


def test_calls_without_rows():
    """Nothing to do is no error, whatever the addresses are."""
    _lib.call("gs_paged_attention", *{**ATTENTION, "num_tokens": 0, "num_seqs": 0, "q": None}.values())
    _lib.call("gs_append_kv", *{**APPEND, "num_tokens": 0, "k": None}.values())
    _lib.call("gs_cache_slots", *{**SLOTS, "num_tokens": 0, "num_seqs": 0, "slots": None}.values())
    _lib.call("gs_residual_norm", *{**NORM, "rows": 0, "x": None, "residual": None}.values())


def test_cpu_tensors_are_refused():
    kc, vc = torch.zeros(4, 2, 16, 64), torch.zeros(4, 2, 16, 64)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)
    q, k = torch.zeros(2, 8, 64), torch.zeros(2, 2, 64)
    with pytest.raises(ValueError, match="on the GPU"):
        paged.paged_attention(q, kc, vc, torch.zeros(2, 1, dtype=torch.int32), i32(1, 1))
    with pytest.raises(ValueError, match="on the GPU"):
        paged.append_kv_(q, k, k, kc, vc, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="on the GPU"):
        paged.cache_slots(torch.zeros(2, 1, dtype=torch.int32), i32(1, 1), 16, 4)
    with pytest.raises(ValueError, match="on the GPU"):
        norms.residual_norm(torch.zeros(2, 8), torch.zeros(2, 8), torch.zeros(8))


def test_registered_shapes():
    with FakeTensorMode():
        i32 = lambda *s: torch.empty(s, dtype=torch.int32, device="cuda")
        t = lambda *s: torch.empty(s, dtype=torch.bfloat16, device="cuda")
        slots, pos = ops.op("cache_slots")(i32(3, 8), i32(3), 16, 24, i32(4), 40)
        assert slots.shape == pos.shape == (40,) and slots.dtype == pos.dtype == torch.int64
        qkv = t(40, 12, 64)
        q = ops.op("append_kv")(qkv[:, :8], qkv[:, 8:10], qkv[:, 10:], t(24, 2, 16, 64), t(24, 2, 16, 64), slots, pos,
                                torch.empty(128, 64, device="cuda"), False)
        assert q.shape == (40, 8, 64) and q.is_contiguous()
        o = ops.op("paged_attention")(qkv[:, :8], t(24, 2, 16, 64), t(24, 2, 16, 64), i32(3, 8), i32(3), i32(4), None, 0, 30)
        assert o.shape == (40, 8, 64) and o.is_contiguous() and o.dtype == torch.bfloat16
        y, r = ops.op("residual_norm")(t(40, 256), torch.empty(40, 256, device="cuda"), t(256), 1e-5, 1.0, None, None, None)
        assert y.dtype == torch.bfloat16 and r.dtype == torch.float32 and y.shape == r.shape == (40, 256)


def test_decoder_arguments():
    lin = lambda n_in, slices, **kw: vllm_layers.SwitchedLoRALinear(
        torch.nn.Linear(n_in, sum(slices), bias=False), 1, 8, num_slices=len(slices), output_slices=slices, **kw)
    one = torch.ones(64)
    args = lambda **kw: {**dict(qkv=lin(64, (128, 64, 64)), o_proj=lin(128, (64,)),
                                gate_up=lin(64, (128, 128), fuse_swiglu=True), down=lin(128, (64,)), input_norm=one,
                                mlp_norm=one, heads=2, kv_heads=1, head_dim=64), **kw}
    decoder.SwitchedDecoderLayer(**args())
    with pytest.raises(ValueError, match="qkv has slices"):
        decoder.SwitchedDecoderLayer(**args(kv_heads=2))
    with pytest.raises(ValueError, match="fuse_swiglu"):
        decoder.SwitchedDecoderLayer(**args(gate_up=lin(64, (128, 128))))
