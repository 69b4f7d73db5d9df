"""What the paged cache's, the norms' and the decoder layer's calls refuse, without a GPU: tangents of forward-mode
differentiation, caches that attention does not take.
"""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode
from torch.autograd import forward_ad

from granite_switch_amd import _lib, decoder, norms, ops, paged, vllm_layers


def _cpu_call():
    """The tensors of a call by name, and the calls that take them."""
    t = dict(q=torch.randn(3, 8, 64), k=torch.randn(3, 2, 64), v=torch.randn(3, 2, 64), kc=torch.randn(4, 2, 16, 64),
             vc=torch.randn(4, 2, 16, 64), rope=torch.randn(8, 64), w=torch.randn(64), x=torch.randn(3, 64), r=torch.randn(3, 64))
    slots, table, lens = torch.arange(3), torch.zeros(3, 4, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    qc = paged.allocate_quantized_cache(4, 2, 16, 64, "cpu")
    return t, {
        "append": (("q", "k", "v", "kc", "vc", "rope"),
                   lambda q, k, v, kc, vc, rope, **_: paged.append_kv_(q, k, v, kc, vc, slots, slots, rope)),
        "append quantised": (("q", "k", "v", "rope", "w"),
                             lambda q, k, v, rope, w, **_: paged.append_kv_(q, k, v, *qc, slots, slots, rope, k_norm=w)),
        "append normed": (("q", "k", "v", "kc", "vc", "w"),
                          lambda q, k, v, kc, vc, w, **_: paged.append_kv_(q, k, v, kc, vc, slots, q_norm=w)),
        "read": (("kc", "vc"), lambda kc, vc, **_: paged.read_kv(kc, vc, slots)),
        "attention": (("q", "kc", "vc"), lambda q, kc, vc, **_: paged.paged_attention(q, kc, vc, table, lens)),
        "attention quantised": (("q",), lambda q, **_: paged.paged_attention(q, *qc, table, lens)),
        "norm": (("x", "r", "w"), lambda x, r, w, **_: norms.residual_norm(x, r, w)),
        "norm, gated": (("x", "w"), lambda x, w, **_: norms.residual_norm(x, x.detach(), w.detach(), gate=w, post_weight=w)),
        "op append": (("q", "k", "v", "w"),
                      lambda q, k, v, w, **_: ops.op("append_kv_normed")(q, k, v, qc[0].values, qc[1].values, qc[0].scales, qc[1].scales,
                                                                         slots, None, None, False, w, w, 1e-5)),
        "op attention": (("q",), lambda q, **_: ops.op("paged_attention_e4m3")(q, qc[0].values, qc[1].values, qc[0].scales, qc[1].scales,
                                                                               table, lens, None, None, 0, None)),
    }


@pytest.mark.parametrize("call", list(_cpu_call()[1]))
def test_tangents_are_refused(call):
    """A dual tensor does not require grad, and its tangent would be dropped without a word."""
    t, calls = _cpu_call()
    takes, run = calls[call]
    for name in takes:
        for no_grad in (False, True):
            with forward_ad.dual_level(), torch.set_grad_enabled(not no_grad):
                args = dict(t)
                args[name] = forward_ad.make_dual(t[name], torch.ones_like(t[name]))
                with pytest.raises(RuntimeError, match="computes no gradients"):
                    run(**args)
    with forward_ad.dual_level(), pytest.raises(ValueError, match="on the GPU"):
        run(**t)                                           # inside a level, but without a tangent


@pytest.mark.parametrize("dim,page,quant", [(40, 16, True), (72, 16, True), (272, 16, True), (64, 12, True), (4, 16, False),
                                            (264, 16, False), (64, 12, False)])
def test_a_layer_refuses_a_cache_that_it_could_not_attend_over(dim, page, quant):
    """Before it stores a row there, not after."""
    lin = lambda n_in, slices, **kw: vllm_layers.SwitchedLoRALinear(
        torch.nn.Linear(n_in, sum(slices), bias=False), 1, 8, num_slices=len(slices), output_slices=slices, **kw)
    one = torch.ones(64)
    layer = decoder.SwitchedDecoderLayer(lin(64, (2 * dim, dim, dim)), lin(2 * dim, (64,)), lin(64, (128, 128), fuse_swiglu=True),
                                         lin(128, (64,)), one, one, 2, 1, dim)
    make = paged.allocate_quantized_cache if quant else paged.allocate_cache
    cache = make(3, 1, page, dim, device="cpu")
    with pytest.raises(ValueError, match=f"head_dim={dim} must be a multiple of {16 if quant else 8}"):
        layer(None, torch.zeros(2, 64), None, cache)
    with pytest.raises(ValueError, match="on the GPU"):
        layer(None, torch.zeros(2, 64), None, make(3, 1, 16, 64, device="cpu"))


@pytest.mark.parametrize("call", ["cache_slots", "residual_norm"])
def test_calls_on_another_device_make_it_the_current_one(monkeypatch, call):
    """A launch, the default stream's among them, goes to the current device, wherever the tensors live."""
    current, launched = [0], []

    class On:
        def __init__(self, device):
            self.index = torch.device(device).index

        def __enter__(self):
            self.was, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.was

    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(_lib, "stream_ptr", lambda device=None: 0)
    monkeypatch.setattr(_lib, "call", lambda name, *args: launched.append((name, current[0])))
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda self: 0)
    monkeypatch.setattr(FakeTensor, "data_ptr", lambda self: 0, raising=False)
    for device in (1, 0, 1):
        with FakeTensorMode(), torch.no_grad():
            t = lambda *s, dtype=torch.float32: torch.empty(s, dtype=dtype, device=f"cuda:{device}")  # noqa: E731
            if call == "cache_slots":
                paged.cache_slots(t(2, 3, dtype=torch.int32), t(2, dtype=torch.int32), 16, 8)
            else:
                norms.residual_norm(t(3, 64), t(3, 64), t(64))
                norms.residual_norm(t(2, 3, 64), t(2, 3, 64), t(64))
        assert launched and all(on == device for _, on in launched), launched
        launched.clear()
        assert current == [0]
