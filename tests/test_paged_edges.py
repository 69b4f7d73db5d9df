"""CPU tests of the paged cache's entry points where a call's arguments, not its sizes, are unusual."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from granite_switch_amd import _lib, decoder, norms, paged, vllm_layers
from test_paged_calls import ATTENTION, P, _refused
from test_paged_model import BF16, FP32, _check_attention

NO_WINDOW = 2 ** 31 - 1                                    # as wide as 32 bits hold


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("window", [NO_WINDOW, NO_WINDOW - 1, NO_WINDOW - 40, 2 ** 31 - 2 ** 16, 2 ** 30])
@pytest.mark.parametrize("n,cached,heads,kv", [([40, 3, 20], [-25, -3, 5], 8, 2), ([200, 1], [-120, 300], 3, 3),
                                               ([7, 1], [-3, 20], 48, 1)])
def test_wide_windows(dtype, window, n, cached, heads, kv):
    """Rows without a position have negative ones: their distance to a wide window's start passes 32 bits."""
    cu = np.concatenate([[0], np.cumsum(n)])
    _check_attention(dtype, np.asarray(n) + np.asarray(cached), cu, heads, kv, 64, 16, window, "heads", cus=16)


def test_rows_and_window_past_32_bits():
    """A table that reaches past a window of nearly 2^31 tokens: only as many rows as leave the sum in 32 bits."""
    change = dict(cu=P, num_tokens=1 << 17, window=(1 << 31) - (1 << 17), max_pages=1 << 27, ld_table=1 << 27)
    e = _refused("gs_paged_attention", ATTENTION, change)
    assert e.status == _lib.GS_ERR_INVALID and "past 32 bits" in str(e)


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (BF16, 128), (BF16, 256), (FP32, 64)])
@pytest.mark.parametrize("cu,rows", [([0, 3, 40], 45), ([0, 0], 7), ([5, 25, 26], 26), ([2, 4], 300), ([0], 9), ([3], 9),
                                     ([0, 4, 9], 9)])
def test_rows_of_no_sequence(dtype, dim, cu, rows):
    """Rows before the first sequence and past the last are written too, every row once."""
    B, heads, kv, page, pages = len(cu) - 1, 6, 2, 16, 8
    lens = np.asarray([cu[s + 1] - cu[s] + 7 for s in range(B)], np.int32)
    table = np.tile(np.arange(4, dtype=np.int32), (max(B, 1), 1))
    cu = np.asarray(cu, np.int32)
    msg, checked = ctypes.create_string_buffer(256), ctypes.c_int64()
    st = (kv * page * dim, page * dim, dim)
    bad = _lib.load().gs_check_paged_addresses(dtype, heads * dim, dim, *st, *st, pages, page, table.ctypes.data, 4, 4,
                                               lens.ctypes.data, cu.ctypes.data, B, rows, heads, kv, dim, 0, heads * dim,
                                               dim, 16, msg, 256, ctypes.byref(checked))
    assert bad == 0, (bad, msg.value.decode() or _lib.last_error())


def test_captured_calls_share_no_workspace(monkeypatch):
    """A graph may be replayed on any stream: what it uses is neither a stream's own buffer nor another graph's."""
    capture = {"id": 0}
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capture["id"] != 0)
    monkeypatch.setattr(_lib, "capture_id", lambda stream: capture["id"], raising=False)
    for name in ("_workspaces", "_captured"):
        monkeypatch.setattr(paged, name, {}, raising=False)
    get = lambda stream, need=1 << 17: paged._workspace(torch.device("cpu"), stream, need)
    eager = get(5)
    assert get(5, 100) is eager and get(6) is not eager
    capture["id"] = 1
    first = get(5)
    assert first is not eager and first.numel() >= 1 << 17
    assert get(5, 100) is first, "the calls of one capture follow each other on its stream"
    assert get(6) is not first, "another stream of the capture may run beside it"
    larger = get(5, 1 << 18)
    assert larger.numel() >= 1 << 18 and get(5) is larger
    capture["id"] = 2
    second = get(5)
    assert second is not eager and second is not first and second is not larger
    capture["id"] = 0
    assert get(5) is eager
    for buf in (eager, first, larger, second):
        assert not buf[: 65536].any(), "counters start at zero"


@pytest.mark.parametrize("captured", [False, True])
def test_only_the_counters_are_cleared(monkeypatch, captured):
    """A workspace is up to tens of megabytes, its counters 64 KB: a graph clears them on every replay."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: captured)
    monkeypatch.setattr(_lib, "capture_id", lambda stream: 3)
    monkeypatch.setattr(paged, "_workspaces", {})
    monkeypatch.setattr(paged, "_captured", {})
    monkeypatch.setattr(torch, "empty", lambda n, **kw: torch.full((n,), 255, **kw))
    buf = paged._workspace(torch.device("cpu"), 5, 1 << 20)
    head = _lib.GS_PAGED_HEAD_BYTES
    assert buf.numel() == 1 << 20 and not buf[:head].any() and bool((buf[head:] == 255).all())


def _tracked():
    """Calls of the entry points, each with one input that autograd tracks; every tensor is on the CPU, which comes later."""
    t = lambda *s: torch.zeros(*s)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)
    slots = torch.zeros(2, dtype=torch.int64)
    attention = dict(q=t(2, 8, 64), k_cache=t(4, 2, 16, 64), v_cache=t(4, 2, 16, 64), page_table=torch.zeros(2, 1, dtype=torch.int32),
                     kv_lens=i32(1, 1))
    append = dict(q=t(2, 8, 64), k=t(2, 2, 64), v=t(2, 2, 64), k_cache=t(4, 2, 16, 64), v_cache=t(4, 2, 16, 64), slots=slots,
                  positions=slots, cos_sin=t(4, 64))
    norm = dict(x=t(2, 64), residual=t(2, 64), weight=t(64), gate=t(2, 64), post_weight=t(64))
    for f, base, names in ((paged.paged_attention, attention, ("q", "k_cache", "v_cache")),
                           (paged.append_kv_, append, ("q", "k", "v", "k_cache", "v_cache", "cos_sin")),
                           (norms.residual_norm, norm, ("x", "residual", "weight", "gate", "post_weight"))):
        for name in names:
            yield pytest.param(f, {**base, name: base[name].clone().requires_grad_()}, id=f"{f.__name__}-{name}")


@pytest.mark.parametrize("f,kw", _tracked())
def test_tracked_inputs_are_refused(f, kw):
    """Nothing here computes gradients: a call that autograd would have to follow says so."""
    with pytest.raises(RuntimeError, match="no gradients"):
        f(**kw)
    with torch.no_grad(), pytest.raises(ValueError, match="on the GPU"):
        f(**kw)


def test_decoder_keeps_norm_weights_out_of_autograd():
    """A model's norm weights are parameters: the decoder, which computes no gradients, takes their values."""
    lin = lambda n_in, slices, **kw: vllm_layers.SwitchedLoRALinear(
        torch.nn.Linear(n_in, sum(slices), bias=False), 1, 8, num_slices=len(slices), output_slices=slices, **kw)
    w = [torch.nn.Parameter(torch.ones(64)) for _ in range(3)]
    layer = decoder.SwitchedDecoderLayer(lin(64, (128, 64, 64)), lin(128, (64,)), lin(64, (128, 128), fuse_swiglu=True),
                                         lin(128, (64,)), w[0], w[1], heads=2, kv_heads=1, head_dim=64)
    dec = decoder.SwitchedDecoder([layer], w[2], 1)
    for got, given in ((layer.input_norm, w[0]), (layer.mlp_norm, w[1]), (dec.final_norm, w[2])):
        assert not got.requires_grad and got.data_ptr() == given.data_ptr()
