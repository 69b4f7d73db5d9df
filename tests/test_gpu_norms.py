"""GPU parity of the fused residual add and norms against a plain float64 form.

Tolerances, u = 2^-24: the sum of h squares is off by a factor within 1 +- h u,
so 1/sqrt by half of that; products and the residual sum add a few u of the
magnitudes they combine; each output is rounded once to its type (bf16 has 8 significant bits: 2^-8).
"""

from __future__ import annotations

import pytest
import torch

from granite_switch_amd import _lib, norms

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF16, FP32 = torch.bfloat16, torch.float32


def _say(msg):
    print(msg, flush=True)


def _reference(x, r, w, eps, scale, gate, post, act):
    """(y, r', magnitude of what r' was summed from, in the scale of y and of r')."""
    rms = lambda t: 1 / (t.pow(2).mean(-1, keepdim=True) + eps).sqrt()  # noqa: E731
    r = r.double()
    mag = r.abs()
    if x is not None:
        b = x.double()
        if post is not None:
            b = b * rms(b) * post.double()
        if gate is not None:
            g = gate.double()
            b = b * (torch.sigmoid(g) if act == "sigmoid" else torch.tanh(g) if act == "tanh" else g)
        mag = mag + (scale * b).abs()
        r = r + scale * b
    inv = rms(r) * w.double()
    return r * inv, r, mag * inv.abs(), mag


def _check(x, r, w, y, ro, eps=1e-5, scale=1.0, gate=None, post=None, act=None):
    want_y, want_r, mag_y, mag_r = _reference(x, r, w, eps, scale, gate, post, act)
    few = (r.shape[-1] + 32) * U
    for name, got, want, mag in (("y", y, want_y, mag_y), ("r", ro, want_r, mag_r)):
        half = 2.0 ** -8 if got.dtype == BF16 else 0.0
        err = (got.double() - want).abs()
        tol = half * want.abs() + 2 * few * mag + 1e-38
        assert bool((err <= tol).all()), (name, float(err.max()), float((err / tol).max()))


@pytest.mark.parametrize("dtype,res", [(BF16, BF16), (BF16, FP32), (FP32, FP32)])
@pytest.mark.parametrize("rows,hidden", [(1, 1), (3, 7), (7, 2048), (5, 4096), (300, 2560), (2, 12800), (9, 1000), (3, 4100),
                                         (2, 16384), (1, 40000), (2, 70000), (65, 64), (4, 520)])
def test_shapes(dev, dtype, res, rows, hidden):
    _say(f"{dtype}/{res} {rows} x {hidden}")
    g = torch.Generator(device=dev).manual_seed(hidden)
    n = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    x, r, w = n(rows, hidden).to(dtype), (3 * n(rows, hidden)).to(res), (1 + 0.1 * n(hidden)).to(dtype)
    post, gate = (1 + 0.1 * n(hidden)).to(dtype), n(rows, hidden).to(dtype)
    for kw in (dict(), dict(post=post), dict(gate=gate, act="sigmoid"), dict(post=post, gate=gate, act="tanh"), dict(gate=gate)):
        y, ro = norms.residual_norm(x, r, w, scale=0.22, gate=kw.get("gate"), post_weight=kw.get("post"), gate_act=kw.get("act"))
        torch.cuda.synchronize()
        _check(x, r, w, y, ro, scale=0.22, **kw)
    # the residual's norm alone
    out = torch.empty(rows, hidden, dtype=dtype, device=dev)
    y, same = norms.residual_norm(None, r, w, out=out)
    torch.cuda.synchronize()
    assert same is r and y is out
    _check(None, r, w, y, r)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("shape", [(5, 256), (5, 1), (256,), (1, 256), (1, 1)])
def test_gate_broadcasts(dev, dtype, shape):
    g = torch.Generator(device=dev).manual_seed(1)
    x, r = (torch.randn(5, 256, generator=g, device=dev).to(dtype) for _ in range(2))
    w = torch.ones(256, device=dev)                       # weights in fp32 beside bf16
    gate = torch.randn(shape, generator=g, device=dev).to(dtype)
    y, ro = norms.residual_norm(x, r, w, gate=gate, gate_act="sigmoid")
    torch.cuda.synchronize()
    _check(x, r, w, y, ro, gate=gate.expand(5, 256), act="sigmoid")
    x3, r3 = x[:4].view(2, 2, 256), r[:4].view(2, 2, 256)
    if shape[0] == 5:
        g3 = gate[:4].view(2, 2, -1)
    else:
        g3 = gate
    y3, ro3 = norms.residual_norm(x3, r3, w, gate=g3, gate_act="sigmoid")
    torch.cuda.synchronize()
    assert torch.equal(y3.view(4, 256), y[:4]) and torch.equal(ro3.view(4, 256), ro[:4])


@pytest.mark.parametrize("hidden", [2048, 100])
def test_in_place_and_strided(dev, hidden):
    g = torch.Generator(device=dev).manual_seed(2)
    buf = torch.randn(40, 3 * hidden, generator=g, device=dev).to(BF16)
    x, r = buf[:, :hidden], buf[:, hidden:2 * hidden]
    w = torch.randn(hidden, generator=g, device=dev).to(BF16)
    x0, r0, rest = x.clone(), r.clone(), buf[:, 2 * hidden:].clone()
    y, ro = norms.residual_norm(x, r, w, scale=0.5, out=x, residual_out=r)
    torch.cuda.synchronize()
    assert y is x and ro is r
    _check(x0, r0, w, y, ro, scale=0.5)
    assert torch.equal(buf[:, 2 * hidden:], rest), "columns outside the outputs were written"


def test_special_rows(dev):
    """A zero row gives zeros (eps > 0); an infinity or NaN stays in its row."""
    x, r, w = torch.zeros(4, 512, device=dev), torch.zeros(4, 512, device=dev), torch.ones(512, device=dev)
    r[1] = torch.randn(512, device=dev)
    r[2, 5], r[3, 7] = float("inf"), float("nan")
    y, ro = norms.residual_norm(x, r, w)
    torch.cuda.synchronize()
    assert bool((y[0] == 0).all()) and bool(torch.isfinite(y[1]).all())
    assert bool(torch.isnan(y[2, 5])) and bool((y[2, :5] == 0).all()) and bool(torch.isnan(y[3]).all())


def test_graph_and_stream(dev):
    x, r, w = torch.randn(33, 4096, device=dev).to(BF16), torch.randn(33, 4096, device=dev).to(BF16), torch.ones(4096, device=dev).to(BF16)
    y, ro = norms.residual_norm(x, r, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gy, gr = norms.residual_norm(x, r, w)
    for _ in range(3):
        x.normal_()
        torch.cuda.synchronize()
        graph.replay()
        y, ro = norms.residual_norm(x, r, w)
        torch.cuda.synchronize()
        assert torch.equal(gy, y) and torch.equal(gr, ro)


def test_refusals(dev):
    x, r, w = torch.randn(4, 64, device=dev), torch.randn(4, 64, device=dev), torch.ones(64, device=dev)
    call = lambda **kw: norms.residual_norm(**{**dict(x=x, residual=r, weight=w), **kw})  # noqa: E731
    call()
    for bad, err in [
        (dict(x=x.half()), (TypeError, ValueError)), (dict(x=x[:3]), ValueError), (dict(residual=r.bfloat16()), TypeError),
        (dict(weight=w[:63]), ValueError), (dict(weight=w.bfloat16()), ValueError), (dict(gate_act="relu"), ValueError),
        (dict(gate=torch.ones(3, 64, device=dev)), RuntimeError), (dict(gate=torch.ones(64, device=dev).half()), TypeError),
        (dict(x=None, gate=x), ValueError), (dict(x=None, post_weight=w), ValueError), (dict(out=x[:3]), ValueError),
        (dict(out=x.bfloat16()), ValueError), (dict(post_weight=w.bfloat16()), ValueError), (dict(x=x.cpu()), ValueError),
        (dict(out=r), _lib.GraniteSwitchError), (dict(residual_out=x), _lib.GraniteSwitchError),
        (dict(eps=-1.0), _lib.GraniteSwitchError), (dict(x=x.t().contiguous().t()), ValueError),
    ]:
        with pytest.raises(err):
            call(**bad)
    big = torch.randn(5, 64, device=dev)
    with pytest.raises(_lib.GraniteSwitchError, match="overlaps"):
        norms.residual_norm(big[:4], r, w, out=big[1:])
    y, ro = norms.residual_norm(x[:0], r[:0], w)
    assert y.shape == ro.shape == (0, 64)
