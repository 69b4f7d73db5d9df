"""What the paged cache's and the norms' calls refuse, without a GPU: tangents of forward-mode differentiation."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from granite_switch_amd import norms, ops, paged


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
