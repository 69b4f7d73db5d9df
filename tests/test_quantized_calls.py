"""CPU tests: what the entry points of a quantised cache and of normed heads refuse, and their ops' shapes.

No kernel is launched: every call here is rejected by its argument checks before any
HIP call, or has no rows.
"""

from __future__ import annotations

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from granite_switch_amd import _lib, decoder, ops, paged, vllm_layers

P = ctypes.c_void_p(4096)                                  # an address that no check reads from
BF16, FP32, E4M3 = _lib.GS_DTYPE_BF16, _lib.GS_DTYPE_FP32, _lib.GS_DTYPE_E4M3

APPEND = dict(dtype=BF16, q=P, q_ts=1024, q_hs=128, k=P, k_ts=256, k_hs=128, v=P, v_ts=256, v_hs=128, num_tokens=2,
              heads=8, kv_heads=2, head_dim=128, q_norm=P, k_norm=P, norm_dtype=BF16, eps=1e-5, positions=P, cos_sin=P,
              max_pos=64, rot_dim=128, interleaved=0, slots=P, cache_dtype=E4M3, k_cache=P, kc_ps=4096, kc_hs=2048,
              kc_rs=128, v_cache=P, vc_ps=4096, vc_hs=2048, vc_rs=128, k_scales=P, ks_ps=32, ks_hs=16, v_scales=P,
              vs_ps=32, vs_hs=16, num_pages=4, page_size=16, q_out=P, o_ts=1024, o_hs=128, stream=None)
READ = dict(dtype=BF16, cache_dtype=E4M3, k_cache=P, kc_ps=4096, kc_hs=2048, kc_rs=128, v_cache=P, vc_ps=4096, vc_hs=2048,
            vc_rs=128, k_scales=P, ks_ps=32, ks_hs=16, v_scales=P, vs_ps=32, vs_hs=16, num_pages=4, page_size=16,
            kv_heads=2, head_dim=128, slots=P, num_tokens=2, k_out=P, ko_ts=256, ko_hs=128, v_out=P, vo_ts=256,
            vo_hs=128, stream=None)
ATTENTION = dict(dtype=BF16, q=P, q_ts=1024, q_hs=128, k=P, k_ps=4096, k_hs=2048, k_rs=128, v=P, v_ps=4096, v_hs=2048,
                 v_rs=128, k_scales=P, ks_ps=32, ks_hs=16, v_scales=P, vs_ps=32, vs_hs=16, num_pages=4, page_size=16,
                 table=P, ld_table=4, max_pages=4, lens=P, cu=None, num_seqs=2, num_tokens=2, max_q=1, heads=8, kv_heads=2,
                 head_dim=128, scale=1.0, window=0, out=P, o_ts=1024, o_hs=128, lse=None, ws=P, ws_bytes=1 << 40,
                 stream=None)


def _refused(name, base, change):
    unknown = set(change) - set(base)
    assert not unknown, unknown
    with pytest.raises(_lib.GraniteSwitchError) as e:
        _lib.call(name, *{**base, **change}.values())
    assert e.value.status == _lib.GS_ERR_INVALID and name in str(e.value)


@pytest.mark.parametrize("change", [
    dict(dtype=7), dict(dtype=E4M3), dict(cache_dtype=FP32), dict(num_tokens=-1), dict(kv_heads=0), dict(head_dim=513),
    dict(rot_dim=130), dict(rot_dim=63), dict(page_size=0), dict(num_pages=0), dict(k=None), dict(v=None), dict(slots=None),
    dict(k_cache=None), dict(v_cache=None), dict(k_scales=None), dict(v_scales=None), dict(q_out=None),
    dict(positions=None), dict(cos_sin=None), dict(max_pos=0), dict(norm_dtype=7), dict(dtype=FP32, norm_dtype=BF16),
    dict(eps=-1.0), dict(eps=float("nan"))], ids=str)
def test_append_arguments(change):
    _refused("gs_append_kv_normed", APPEND, change)


def test_more_rows_than_a_launch_has():
    _refused("gs_append_kv_normed", APPEND, dict(num_tokens=2 ** 31 - 1, q_ts=4096, heads=32, head_dim=512, q_hs=512, k_hs=512,
                                                 v_hs=512, o_hs=512))
    _refused("gs_append_kv_normed", APPEND, dict(num_tokens=2 ** 27))         # 2.5 x 2^23 workgroups of 256 threads
    _refused("gs_read_kv", READ, dict(num_tokens=2 ** 25, kv_heads=16, ko_ts=2048, vo_ts=2048))


def test_more_pages_than_an_id_counts():
    for name, base in (("gs_append_kv_normed", APPEND), ("gs_read_kv", READ)):
        _refused(name, base, dict(num_pages=2 ** 31))


@pytest.mark.parametrize("change", [
    dict(dtype=7), dict(dtype=E4M3), dict(cache_dtype=FP32), dict(num_tokens=-1), dict(kv_heads=0), dict(head_dim=513),
    dict(page_size=0), dict(num_pages=0), dict(slots=None), dict(k_cache=None), dict(v_cache=None), dict(k_scales=None),
    dict(v_scales=None), dict(k_out=None), dict(v_out=None)], ids=str)
def test_read_arguments(change):
    _refused("gs_read_kv", READ, change)


@pytest.mark.parametrize("change", [
    dict(dtype=7), dict(num_tokens=-1), dict(num_tokens=3), dict(heads=7), dict(kv_heads=0), dict(head_dim=272),
    dict(head_dim=104), dict(page_size=12), dict(num_pages=0), dict(ld_table=3), dict(window=-1), dict(q=None), dict(k=None),
    dict(out=None), dict(lens=None), dict(k_scales=None), dict(v_scales=None), dict(k_scales=ctypes.c_void_p(4100)),
    dict(vs_hs=12), dict(k=ctypes.c_void_p(4104)), dict(k_rs=136), dict(v_rs=-128), dict(o_ts=1028)], ids=str)
def test_attention_arguments(change):
    _refused("gs_paged_attention_e4m3", ATTENTION, change)


def test_calls_without_rows():
    """Nothing to do is no error, whatever the addresses are."""
    _lib.call("gs_append_kv_normed", *{**APPEND, "num_tokens": 0, "k": None}.values())
    _lib.call("gs_read_kv", *{**READ, "num_tokens": 0, "k_out": None}.values())
    _lib.call("gs_paged_attention_e4m3", *{**ATTENTION, "num_tokens": 0, "num_seqs": 0, "q": None}.values())


def _cache(pages=4, kv=2, page=16, dim=64, device="cuda"):
    return paged.allocate_quantized_cache(pages, kv, page, dim, device)


def test_cpu_tensors_are_refused():
    kc, vc = _cache(device="cpu")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)
    q, k, slots = torch.zeros(2, 8, 64), torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="on the GPU"):
        paged.paged_attention(q, kc, vc, torch.zeros(2, 1, dtype=torch.int32), i32(1, 1))
    with pytest.raises(ValueError, match="on the GPU"):
        paged.append_kv_(q, k, k, kc, vc, slots)
    with pytest.raises(ValueError, match="on the GPU"):
        paged.append_kv_(q, k, k, k.new_zeros(4, 2, 16, 64), k.new_zeros(4, 2, 16, 64), slots, q_norm=torch.ones(64))
    with pytest.raises(ValueError, match="on the GPU"):
        paged.read_kv(kc, vc, slots)


def test_python_refusals(monkeypatch):
    """The checks of shapes, types and layouts, on tensors without memory."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    with FakeTensorMode(), torch.no_grad():
        t = lambda *s, dtype=torch.bfloat16: torch.empty(s, dtype=dtype, device="cuda:0")
        i32 = lambda *s: t(*s, dtype=torch.int32)
        q, k, slots = t(3, 8, 64), t(3, 2, 64), t(3, dtype=torch.int64)
        kc, vc = _cache(device="cuda:0")
        plain = t(4, 2, 16, 64)
        append = lambda kc=kc, vc=vc, q=q, k=k, **kw: paged.append_kv_(q, k, k, kc, vc, slots, **kw)
        with pytest.raises(ValueError, match="one cache is quantised"):
            append(vc=plain)
        with pytest.raises(ValueError, match="float8_e4m3fn"):
            append(kc=paged.QuantizedCache(plain, kc.scales))
        with pytest.raises(ValueError, match="scales"):
            append(kc=paged.QuantizedCache(kc.values, t(4, 2, 16)))
        with pytest.raises(ValueError, match="scales"):
            append(vc=paged.QuantizedCache(vc.values, vc.scales[:, :, :8]))
        with pytest.raises(ValueError, match="side by side"):
            append(kc=paged.QuantizedCache(kc.values, t(4, 16, 2, dtype=torch.float8_e8m0fnu).permute(0, 2, 1)))
        with pytest.raises(ValueError, match="bfloat16"):
            append(kc=plain.float(), vc=plain.float(), q_norm=t(64))
        with pytest.raises(ValueError, match="q_norm must be"):
            append(q_norm=t(63))
        with pytest.raises(ValueError, match="k_norm must be"):
            append(k_norm=t(64, dtype=torch.float16))
        with pytest.raises(ValueError, match="k_norm must be"):
            append(k_norm=t(64, 2)[:, 0])
        with pytest.raises(ValueError, match="q_norm is"):
            append(q_norm=t(64), k_norm=t(64, dtype=torch.float32))
        with pytest.raises(ValueError, match="q_norm without q"):
            append(q=None, q_norm=t(64))
        with pytest.raises(TypeError, match="unsupported dtype"):
            append(k=k.half())
        far = 2 ** 32 + 2                                  # 2 in 32 bits
        with pytest.raises(ValueError, match="heads of 64"):
            append(q=t(1, 1, 64).expand(3, far, 64))
        with pytest.raises(ValueError, match="heads of 64"):
            append(k=t(1, 1, 64).expand(3, far, 64))
        with pytest.raises(ValueError, match="pages of"):
            paged.read_kv(t(4, 1, 16, 64).expand(4, far, 16, 64), t(4, 1, 16, 64).expand(4, far, 16, 64), slots)
        read = lambda kc=kc, vc=vc, slots=slots, **kw: paged.read_kv(kc, vc, slots, **kw)
        with pytest.raises(TypeError, match="unsupported dtype"):
            read(dtype=torch.float16)
        with pytest.raises(ValueError, match="slots"):
            read(slots=i32(3))
        with pytest.raises(ValueError, match="k_out"):
            read(k_out=t(3, 2, 32))
        with pytest.raises(ValueError, match="k_cache must be"):
            read(kc=plain, vc=plain, dtype=torch.float32)
        with pytest.raises(ValueError, match="one cache is quantised"):
            read(kc=plain)
        with pytest.raises(ValueError, match="float8_e4m3fn"):
            paged.paged_attention(q, paged.QuantizedCache(plain, kc.scales), vc, i32(3, 4), i32(3))
        with pytest.raises(ValueError, match="one cache is quantised"):
            paged.paged_attention(q, kc, plain, i32(3, 4), i32(3))


def test_tracked_inputs_are_refused(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    with FakeTensorMode():
        q, k = (torch.empty(3, h, 64, dtype=torch.bfloat16, device="cuda:0") for h in (8, 2))
        kc, vc = _cache(device="cuda:0")
        w = torch.nn.Parameter(torch.empty(64, dtype=torch.bfloat16, device="cuda:0"))
        slots = torch.empty(3, dtype=torch.int64, device="cuda:0")
        with pytest.raises(RuntimeError, match="computes no gradients"):
            paged.append_kv_(q, k, k, kc, vc, slots, k_norm=w)
        with pytest.raises(RuntimeError, match="computes no gradients"):
            paged.append_kv_(q.requires_grad_(), k, k, kc, vc, slots)


def test_registered_shapes():
    with FakeTensorMode():
        i32 = lambda *s: torch.empty(s, dtype=torch.int32, device="cuda")
        t = lambda *s: torch.empty(s, dtype=torch.bfloat16, device="cuda")
        kc, vc = _cache(24)
        slots = torch.empty(40, dtype=torch.int64, device="cuda")
        rope = torch.empty(128, 64, device="cuda")
        qkv = t(40, 12, 64)
        args = (qkv[:, :8], qkv[:, 8:10], qkv[:, 10:])
        q = ops.op("append_kv_normed")(*args, kc.values, vc.values, kc.scales, vc.scales, slots, slots, rope, False, t(64),
                                       t(64), 1e-5)
        assert q.shape == (40, 8, 64) and q.is_contiguous()
        q = ops.op("append_kv_normed")(*args, t(24, 2, 16, 64), t(24, 2, 16, 64), None, None, slots, slots, rope, False, t(64),
                                       None, 1e-5)
        assert q.shape == (40, 8, 64)
        k, v = ops.op("read_kv")(kc.values, vc.values, kc.scales, vc.scales, slots, torch.float32)
        assert k.shape == v.shape == (40, 2, 64) and k.dtype == torch.float32
        k, v = ops.op("read_kv")(kc.values, vc.values, kc.scales, vc.scales, slots, None)
        assert k.dtype == torch.bfloat16
        o = ops.op("paged_attention_e4m3")(args[0], kc.values, vc.values, kc.scales, vc.scales, i32(3, 8), i32(3), i32(4), None, 0, 30)
        assert o.shape == (40, 8, 64) and o.is_contiguous() and o.dtype == torch.bfloat16


def test_decoder_norms():
    lin = lambda n_in, slices, **kw: vllm_layers.SwitchedLoRALinear(
        torch.nn.Linear(n_in, sum(slices), bias=False), 1, 8, num_slices=len(slices), output_slices=slices, **kw)
    one = torch.ones(64)
    args = dict(qkv=lin(64, (128, 64, 64)), o_proj=lin(128, (64,)), gate_up=lin(64, (128, 128), fuse_swiglu=True),
                down=lin(128, (64,)), input_norm=one, mlp_norm=one, heads=2, kv_heads=1, head_dim=64)
    layer = decoder.SwitchedDecoderLayer(**args, q_norm=torch.nn.Parameter(one), k_norm=one)
    assert not layer.q_norm.requires_grad and "q_norm" in dict(layer.named_buffers())
    assert decoder.SwitchedDecoderLayer(**args).q_norm is None
    with pytest.raises(ValueError, match="k_norm"):
        decoder.SwitchedDecoderLayer(**args, k_norm=torch.ones(32))
