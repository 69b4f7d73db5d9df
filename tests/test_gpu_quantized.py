"""GPU parity of the quantised paged cache: append with norms, read, attention, and the decoder over it.

References are plain float64 restatements.  Tolerances, with u = 2^-24 (fp32) and
2^-8 for a rounding to bf16:

  norm      a sum of D squares, its product, rsqrt, two products: (D / 2 + 8) u relative
  rotation  a c - b s in fp32: 4 u (|a| + |b|)
  e4m3      half a step, 2^-4 of the value, or 2^-10 of the scale where that is more; the
            scale is the reference's unless the row's maximum is within those errors of 448
            times a power of two.  Without norm and rotation: equal, bit for bit.
  attention as in test_gpu_paged.py: keys and values are exact in bf16 and fp32, a
            probability times its value's scale is rounded once, as a probability is there.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from granite_switch_amd import _lib, decoder, ops, paged, vllm_layers
from test_gpu_paged import Batch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF16, FP32 = torch.bfloat16, torch.float32
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _say(msg):
    print(msg, flush=True)


def _bytes(t):
    return t.view(torch.uint8)


def exponents(x):
    """The least e >= -126 with |row| <= 448 2^e, of rows of finite float64."""
    m, e = torch.frexp(x.abs().amax(-1))
    return torch.where(m > 0, torch.where(m <= 0.875, e - 9, e - 8), -126).clamp(min=-126)


def quantise(x):
    """(e4m3, e8m0) of the rows of x: the product with a power of two is exact, torch's cast rounds to nearest even."""
    e = exponents(x.double())
    y = (x.double() * torch.exp2(-e.double())[..., None]).float()
    return y.to(E4M3), (e + 127).to(torch.uint8).view(E8M0)


def held(values, scales):
    """Rows as float64."""
    return values.double() * torch.exp2(_bytes(scales).double() - 127)[..., None]


def make_cache(dev, pages, kv, page, dim, layout="heads", junk=True):
    """A quantised cache whose rows are NaN with NaN scales, in an order of its dimensions."""
    shape = (pages, kv, page, dim) if layout == "heads" else (pages, page, kv, dim)
    values = torch.empty(shape, dtype=torch.uint8, device=dev)
    scales = torch.empty((pages, kv, page), dtype=torch.uint8, device=dev)
    if junk:
        values.fill_(0x7F)
        scales.fill_(0xFF)
    values = values.view(E4M3)
    return paged.QuantizedCache(values if layout == "heads" else values.permute(0, 2, 1, 3), scales.view(E8M0))


# ---------------------------------------------------------------------------
# Append
# ---------------------------------------------------------------------------
def _normed(x, w, eps):
    """float64 rows and the relative error that fp32 leaves in them."""
    x = x.double()
    if w is None:
        return x, 0.0
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double(), (x.shape[-1] / 2 + 8) * U


def _turned(x, rel, table, pos, interleaved):
    """Rotated float64 rows and their error's bound."""
    err = rel * x.abs()
    if table is None:
        return x, err
    R = table.shape[1]
    c, s = (t[:, None, :] for t in table.double()[pos].chunk(2, -1))
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., : R // 2], x[..., R // 2:R])
    lim = (rel + 4 * U) * (a.abs() + b.abs())
    out, err = x.clone(), err.clone()
    for o, v in ((out, (a * c - b * s, b * c + a * s)), (err, (lim, lim))):
        if interleaved:
            o[..., 0:R:2], o[..., 1:R:2] = v
        else:
            o[..., : R // 2], o[..., R // 2:R] = v
    return out, err


def _check_rounded(got, want, err, dtype):
    tol = err * 1.01 + want.abs() * (2.0 ** -8 if dtype == BF16 else U) + 1e-38
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())


def _check_quantised(values, scales, want, err):
    top, slack = want.abs().amax(-1), err.amax(-1)
    e = _bytes(scales).double() - 127
    lo, hi = exponents((top - slack).clamp(min=0)[..., None]), exponents((top + slack)[..., None])
    assert bool(((e >= lo) & (e <= hi)).all())
    unit = torch.exp2(e)[..., None]
    tol = torch.maximum((want.abs() + err) * 2.0 ** -4, unit * 2.0 ** -10) + err * 1.01
    off = (held(values, scales) - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())


def _append_case(dev, dtype, T, H, HK, D, R, page, layout, interleaved, quant, qn, kn, wtype, seed, cols=0, sizes=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = np.random.default_rng(seed)
    rows = (torch.randn(T, (H + 2 * HK) * D + cols, generator=g, device=dev)
            * torch.exp(sizes * torch.randn(T, 1, generator=g, device=dev))).to(dtype)
    q, k, v = (rows[:, a * D + cols: b * D + cols].unflatten(1, (-1, D)) for a, b in ((0, H), (H, H + HK), (H + HK, H + 2 * HK)))
    pages = -(-T // page) + 2
    slots = rng.permutation(pages * page)[:T]
    slots[rng.random(T) < 0.1] = rng.choice([-1, -7, pages * page, 2 ** 40])
    slots = torch.tensor(slots, device=dev)
    weight = lambda: (1 + 0.3 * torch.randn(D, generator=g, device=dev)).to(wtype)  # noqa: E731
    q_norm, k_norm = weight() if qn else None, weight() if kn else None
    table = paged.rope_table(300, R, device=dev) if R else None
    pos = torch.randint(0, 300, (T,), generator=g, device=dev)
    if quant:
        caches = [make_cache(dev, pages, HK, page, D, layout) for _ in range(2)]
        before = [(_bytes(c.values).clone(), _bytes(c.scales).clone()) for c in caches]
    else:
        caches = [torch.full((pages, HK, page, D) if layout == "heads" else (pages, page, HK, D), 7.0, dtype=dtype, device=dev)
                  for _ in range(2)]
        caches = caches if layout == "heads" else [c.permute(0, 2, 1, 3) for c in caches]
        before = [c.clone() for c in caches]
    eps = 1e-5
    got = paged.append_kv_(q, k, v, *caches, slots, pos, table, interleaved=interleaved, q_norm=q_norm, k_norm=k_norm, eps=eps)
    kept = (slots >= 0) & (slots < pages * page)
    at = slots[kept]
    if H:
        _check_rounded(got, *_turned(*_normed(q, q_norm, eps), table, pos, interleaved), dtype)
    for c, b, rows, w, turn in ((caches[0], before[0], k, k_norm, table), (caches[1], before[1], v, None, None)):
        want, err = _turned(*_normed(rows, w, eps), turn, pos, interleaved)
        want, err = want[kept], err.expand_as(want)[kept]
        untouched = torch.ones(pages * page, dtype=torch.bool, device=dev)
        untouched[at] = False
        if quant:
            values, scales = _bytes(c.values)[at // page, :, at % page], _bytes(c.scales)[at // page, :, at % page]
            if w is None and turn is None:
                y, s = quantise(want)
                assert torch.equal(scales, _bytes(s)) and torch.equal(values.view(E4M3).float(), y.float())
            else:
                _check_quantised(values.view(E4M3), scales.view(E8M0), want, err)
            for x, y in zip(c, b):
                rest = _bytes(x).transpose(1, 2).flatten(0, 1)[untouched]
                assert torch.equal(rest, y.transpose(1, 2).flatten(0, 1)[untouched]), "rows of no token were written"
        else:
            _check_rounded(c[at // page, :, at % page], want, err, dtype)
            assert torch.equal(c.transpose(1, 2).flatten(0, 1)[untouched], b.transpose(1, 2).flatten(0, 1)[untouched])


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("T,H,HK,D,R,page,layout,interleaved,qn,kn,cols", [
    (1, 4, 1, 128, 128, 16, "heads", False, True, True, 0),
    (37, 32, 8, 128, 128, 16, "heads", False, True, True, 0),
    (700, 8, 2, 128, 64, 64, "tokens", True, False, True, 0),
    (65, 6, 3, 80, 80, 24, "heads", False, True, True, 8),
    (65, 6, 3, 80, 16, 24, "tokens", True, True, False, 0),
    (33, 2, 2, 512, 512, 8, "heads", False, True, True, 0),
    (33, 2, 1, 256, 128, 7, "heads", False, True, True, 16),
    (50, 3, 3, 64, 64, 1, "tokens", False, True, True, 0),
    (41, 5, 2, 58, 10, 5, "heads", False, True, True, 0),       # element by element
    (41, 5, 2, 128, 128, 16, "heads", True, True, True, 3),     # the same, for its alignment
    (29, 2, 1, 301, 300, 16, "tokens", True, True, True, 0),
    (20, 0, 4, 64, 64, 16, "heads", False, False, True, 0),     # no queries
    (90, 4, 2, 1, 0, 16, "heads", False, True, True, 0),
])
def test_append(dev, dtype, quant, T, H, HK, D, R, page, layout, interleaved, qn, kn, cols):
    _say(f"append {dtype} quant={quant} T={T} {H}+{HK}x{D} rot {R} page {page} {layout} pairs={interleaved} offset {cols}")
    for i, wtype in enumerate({dtype, FP32}):
        _append_case(dev, dtype, T, H, HK, D, R, page, layout, interleaved, quant, qn, kn, wtype, seed=T + D + i, cols=cols)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_append_without_norms(dev, dtype):
    _say(f"append quantised, no norms {dtype}")
    _append_case(dev, dtype, 129, 8, 4, 128, 128, 16, "heads", False, True, False, False, dtype, seed=1)
    _append_case(dev, dtype, 129, 8, 4, 96, 0, 40, "tokens", False, True, False, False, dtype, seed=2, sizes=20.0)
    _append_case(dev, dtype, 600, 2, 4, 30, 0, 16, "heads", False, True, False, False, dtype, seed=3, sizes=20.0)


@pytest.mark.parametrize("dim", [128, 33])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_append_extremes(dev, dtype, dim):
    """Zeros, the ends of the types' ranges, powers of two around 448, ties, and what is not finite."""
    _say(f"append extremes {dtype} {dim}")
    big = torch.finfo(dtype).max
    rows = [torch.zeros(dim), torch.full((dim,), big / 2), torch.full((dim,), 1e-38), torch.full((dim,), 2.0 ** -133)]
    for top in (448.0, 449.0 if dtype == FP32 else 450.0, 447.0, 240.0, 256.0, 1.75, 1.7578125, 7.0 * 2.0 ** -130, 2.0 ** -140):
        rows.append(torch.linspace(-1, 1, dim) * top * 0.99)
        rows[-1][dim // 3] = top
    steps = torch.arange(dim) % 32                        # halves of steps: ties
    rows.append((1 + (2 * steps + 1) / 16.0) * 2.0 ** (torch.arange(dim) % 20 - 12.0))
    rows[-1][0] = 448.0
    k = torch.stack(rows).to(dtype).to(dev)[:, None, :]
    T = k.shape[0]
    kc, vc = (make_cache(dev, 3, 1, 16, dim) for _ in range(2))
    slots = torch.arange(T, device=dev)
    paged.append_kv_(None, k, -k, kc, vc, slots)
    y, s = quantise(k)
    for c, sign in ((kc, 1), (vc, -1)):
        assert torch.equal(_bytes(c.scales)[slots // 16, :, slots % 16], _bytes(s))
        assert torch.equal(_bytes(c.values)[slots // 16, :, slots % 16].view(E4M3).float(), sign * y.float())
    # one value of a row that is not finite becomes NaN, the others are as without it
    for bad in (math.inf, -math.inf, math.nan):
        odd = k.clone()
        odd[:, 0, 1] = bad
        paged.append_kv_(None, odd, odd, kc, vc, slots)
        rest = k.clone()
        rest[:, 0, 1] = 0
        y, s = quantise(rest)
        assert torch.equal(_bytes(kc.scales)[slots // 16, :, slots % 16], _bytes(s))
        got = _bytes(vc.values)[slots // 16, :, slots % 16].view(E4M3).float()
        assert bool(got[:, 0, 1].isnan().all())
        got[:, 0, 1] = 0
        assert torch.equal(got, y.float())


@pytest.mark.parametrize("dim", [128, 33])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("quant", [True, False])
def test_norms_of_rows_that_are_not_finite(dev, quant, dtype, dim):
    """x / sqrt(mean(x^2) + eps): an infinity gives NaN beside zeros, a NaN gives NaN everywhere; other heads as without."""
    _say(f"norms, not finite {dtype} quant={quant} {dim}")
    g = torch.Generator(device=dev).manual_seed(7)
    x = torch.randn(9, 4, dim, generator=g, device=dev).to(dtype)
    w = (1 + 0.3 * torch.randn(dim, generator=g, device=dev)).to(dtype)
    slots = torch.arange(9, device=dev)

    def run(x):
        caches = make_cache(dev, 1, 4, 16, dim), make_cache(dev, 1, 4, 16, dim)
        if not quant:
            caches = [torch.zeros(1, 4, 16, dim, dtype=dtype, device=dev) for _ in range(2)]
        q = paged.append_kv_(x, x, x, *caches, slots, q_norm=w, k_norm=w)
        return q, paged.read_kv(*caches, slots, FP32 if quant else None)[0]

    plain = run(x)
    for bad in (math.inf, -math.inf, math.nan):
        odd = x.clone()
        odd[3, 1, 2] = bad
        for got, want in zip(run(odd), plain):
            want = want.clone()
            want[3, 1] = math.nan if math.isnan(bad) else 0.0
            want[3, 1, 2] = math.nan
            assert torch.equal(got.isnan(), want.isnan())
            assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


def test_eps_by_value(dev):
    """An eps that is a tensor, or an int, counts as the number it holds at the call."""
    x = torch.randn(5, 2, 64, generator=torch.Generator(device=dev).manual_seed(8), device=dev)
    w, slots = torch.ones(64, device=dev), torch.full((5,), -1, device=dev)
    caches = paged.allocate_cache(1, 2, 16, 64, FP32, dev)
    run = lambda eps: paged.append_kv_(x, x, x, *caches, slots, q_norm=w, eps=eps)  # noqa: E731
    eps = torch.tensor(1e-5)
    assert torch.equal(run(eps), run(1e-5))
    eps.fill_(2.0)
    assert torch.equal(run(eps), run(2)) and not torch.equal(run(2.0), run(1e-5))


def test_append_in_place_and_strided(dev):
    _say("append in place, scales with strides of their own")
    g = torch.Generator(device=dev).manual_seed(4)
    T, H, HK, D, page, pages = 45, 6, 3, 64, 16, 4
    qkv = torch.randn(T, H + 2 * HK, D, generator=g, device=dev).to(BF16)
    w = torch.randn(D, generator=g, device=dev).to(BF16)
    slots = torch.randperm(pages * page, generator=g, device=dev)[:T]
    pos, table = torch.arange(T, device=dev), paged.rope_table(64, D, device=dev)
    one = [make_cache(dev, pages, HK, page, D) for _ in range(2)]
    # heads and pages further apart, more rows than the page has
    big = torch.full((pages + 1, HK + 2, 2 * page), 9, dtype=torch.uint8, device=dev)
    two = [paged.QuantizedCache(make_cache(dev, pages, HK, page, D, "tokens").values,
                                big[i:, i:][:pages, :HK, i * page:(i + 1) * page].view(E8M0) if i == 0 else
                                torch.full((pages, HK, page), 9, dtype=torch.uint8, device=dev).view(E8M0)) for i in range(2)]
    a = paged.append_kv_(qkv[:, :H], qkv[:, H:H + HK], qkv[:, H + HK:], *one, slots, pos, table, q_norm=w, k_norm=w)
    q = qkv[:, :H]
    b = paged.append_kv_(q, qkv[:, H:H + HK], qkv[:, H + HK:], *two, slots, pos, table, q_out=q, q_norm=w, k_norm=w)
    assert b is q and torch.equal(a, b)
    for x, y in zip(one, two):
        at = (slots // page, slice(None), slots % page)
        assert torch.equal(_bytes(x.values)[at], _bytes(y.values)[at]) and torch.equal(_bytes(x.scales)[at], _bytes(y.scales)[at])
    written = torch.zeros_like(big, dtype=torch.bool)
    written[:pages, :HK, :page] = True
    assert bool((big[~written] == 9).all())
    for kv in ((paged.read_kv(*one, slots), paged.read_kv(*two, slots))):
        assert torch.equal(kv[0], paged.read_kv(*one, slots)[0])


def test_calls_without_rows(dev):
    _say("calls without rows")
    kc, vc = (make_cache(dev, 2, 2, 16, 64) for _ in range(2))
    none = torch.empty(0, dtype=torch.int64, device=dev)
    q, k = torch.empty(0, 8, 64, dtype=BF16, device=dev), torch.empty(0, 2, 64, dtype=BF16, device=dev)
    w = torch.ones(64, dtype=BF16, device=dev)
    for caches in ((kc, vc), (torch.zeros(2, 2, 16, 64, dtype=BF16, device=dev),) * 2):
        out = paged.append_kv_(q, k, k, *caches, none, none, paged.rope_table(8, 64, device=dev), q_norm=w, k_norm=w)
        assert out.shape == q.shape
        assert all(x.shape == (0, 2, 64) and x.dtype == BF16 for x in paged.read_kv(*caches, none))
    out = paged.paged_attention(q, kc, vc, torch.empty(0, 1, dtype=torch.int32, device=dev),
                                torch.empty(0, dtype=torch.int32, device=dev))
    assert out.shape == q.shape
    assert bool((_bytes(kc.values) == 0x7F).all()) and bool((_bytes(kc.scales) == 0xFF).all())


def test_results_are_contiguous_whatever_the_inputs(dev):
    """Queries in another order of their dimensions: new results are [T, heads, D] in memory."""
    _say("permuted inputs")
    g = torch.Generator(device=dev).manual_seed(8)
    T, H, HK, D = 33, 6, 3, 64
    q = torch.randn(H, T, D, generator=g, device=dev).to(BF16).transpose(0, 1)
    k, v = (torch.randn(HK, T, D, generator=g, device=dev).to(BF16).transpose(0, 1) for _ in range(2))
    slots, pos, rope = torch.arange(T, device=dev), torch.arange(T, device=dev), paged.rope_table(64, D, device=dev)
    w = torch.randn(D, generator=g, device=dev).to(BF16)
    res = []
    for args in ((q, k, v), (q.contiguous(), k.contiguous(), v.contiguous())):
        caches = [make_cache(dev, 3, HK, 16, D) for _ in range(2)]
        out = paged.append_kv_(*args, *caches, slots, pos, rope, q_norm=w, k_norm=w)
        o = paged.paged_attention(args[0], *caches, torch.arange(3, dtype=torch.int32, device=dev)[None],
                                  torch.tensor([T], dtype=torch.int32, device=dev), torch.tensor([0, T], dtype=torch.int32, device=dev))
        assert out.is_contiguous() and o.is_contiguous()
        res.append((out, o, *paged.read_kv(*caches, slots)))
    assert all(torch.equal(a, b) for a, b in zip(*res))


# ---------------------------------------------------------------------------
# Read
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("T,HK,D,page,layout", [(1, 1, 16, 1, "heads"), (257, 8, 128, 16, "heads"), (300, 3, 80, 24, "tokens"),
                                                (77, 2, 512, 5, "heads"), (130, 5, 64, 64, "tokens"), (90, 2, 33, 16, "heads"),
                                                (40, 33, 8, 16, "tokens"), (9, 4096, 16, 2, "heads")])
def test_read(dev, dtype, T, HK, D, page, layout):
    _say(f"read {dtype} T={T} {HK}x{D} page {page} {layout}")
    g = torch.Generator(device=dev).manual_seed(T)
    pages = T // page + 2
    kc, vc = (make_cache(dev, pages, HK, page, D, layout) for _ in range(2))
    for c in (kc, vc):                                     # every byte: subnormals, NaN, both zeros, every scale
        _bytes(c.values).copy_(torch.randint(0, 256, c.values.shape, generator=g, device=dev).to(torch.uint8))
        _bytes(c.scales).copy_(torch.randint(20 if dtype == BF16 else 0, 240, c.scales.shape, generator=g, device=dev).to(torch.uint8))
    slots = torch.randint(-3, pages * page + 3, (T,), generator=g, device=dev)
    slots[T // 2:] = slots[: T - T // 2].clone()           # the same slot again
    got = paged.read_kv(kc, vc, slots, dtype)
    live = (slots >= 0) & (slots < pages * page)
    at = slots.clamp(0, pages * page - 1)
    for x, c in zip(got, (kc, vc)):
        y = _bytes(c.values)[at // page, :, at % page].view(E4M3)
        want = torch.where(live[:, None, None], held(y, _bytes(c.scales)[at // page, :, at % page].view(E8M0)), 0.0)
        assert x.dtype == dtype and torch.equal(x.double().isnan(), want.isnan())
        assert torch.equal(x.double().nan_to_num(0.0), want.nan_to_num(0.0))
    # into views, with a row between the heads
    out = torch.full((T, 2 * HK, 2 * D + 3), 5.0, dtype=dtype, device=dev)
    ko, vo = out[:, :HK, :D], out[:, HK:, D:2 * D]
    again = paged.read_kv(kc, vc, slots, dtype, ko, vo)
    assert again[0] is ko and torch.equal(ko.isnan(), got[0].isnan()) and torch.equal(vo.nan_to_num(0.0), got[1].nan_to_num(0.0))
    assert bool((out[:, :HK, D:] == 5).all()) and bool((out[:, HK:, :D] == 5).all())


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("D", [64, 7])
def test_read_of_a_plain_cache(dev, dtype, D):
    _say(f"read of a plain cache {dtype} {D}")
    kc, vc = (torch.randn(5, 3, 16, D, device=dev).to(dtype) for _ in range(2))
    slots = torch.tensor([0, 79, -1, 80, 17, 17], device=dev)
    k, v = paged.read_kv(kc, vc, slots)
    assert k.dtype == dtype
    for x, c in ((k, kc), (v, vc)):
        rows = c.transpose(1, 2).flatten(0, 1)
        assert torch.equal(x[[0, 1, 4, 5]], rows[[0, 79, 17, 17]]) and bool((x[2:4] == 0).all())


def test_far_slots(dev):
    """Slots and pages whose offsets pass 32 bits."""
    _say("append, read and attention past 4 GiB of a cache")
    HK, D, page = 8, 256, 64
    pages = (1 << 32) // (HK * D * page) + 9
    kc, vc = (make_cache(dev, pages, HK, page, D, junk=False) for _ in range(2))
    for c in (kc, vc):
        _bytes(c.values)[0].fill_(0x7F)
        _bytes(c.values)[-8:].fill_(0x7F)
    g = torch.Generator(device=dev).manual_seed(5)
    L = 100
    table = torch.tensor([[pages - 3, pages - 1]], dtype=torch.int32, device=dev)
    lens = torch.tensor([L], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, L], dtype=torch.int32, device=dev)
    slots, _ = paged.cache_slots(table, lens, page, pages, cu, L)
    k, v = (torch.randn(L, HK, D, generator=g, device=dev).to(BF16) for _ in range(2))
    paged.append_kv_(None, k, v, kc, vc, slots)
    got = paged.read_kv(kc, vc, slots, FP32)
    for x, y in zip(got, (k, v)):
        assert torch.equal(x.double(), held(*quantise(y)))
    q = torch.randn(L, HK, D, generator=g, device=dev).to(BF16)
    o = paged.paged_attention(q, kc, vc, table, lens, cu)
    s = torch.einsum("thd,jhd->htj", q.double().cpu(), got[0].double().cpu()) / 16
    s = s.masked_fill(torch.ones(L, L, dtype=torch.bool).triu(1), -math.inf)
    want = torch.einsum("htj,jhd->thd", torch.softmax(s, -1), got[1].double().cpu())
    assert (o.double().cpu() - want).abs().max() < 2.0 ** -7 * 1.01 * got[1].abs().max()


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
class QBatch(Batch):
    """A batch whose cache is quantised: the rows compared with are what it holds, the others NaN with NaN scales."""

    def __init__(self, dev, n, cached, heads, kv, dim, page=16, dtype=BF16, layout="heads", seed=0, decode=False, spread=1.0):
        super().__init__(dev, n, cached, heads, kv, dim, page, FP32, layout, seed, decode)
        g = torch.Generator(device=dev).manual_seed(seed + 1)
        self.dtype, self.q = dtype, self.q.to(dtype)
        pages = self.k.shape[0]
        caches = []
        for rows in self.rows:
            c = make_cache(dev, pages, kv, page, dim, layout)
            for s, x in enumerate(rows):
                if x.shape[0] == 0:
                    continue
                x = x * torch.exp(spread * torch.randn(x.shape[:2], generator=g, device=dev))[..., None]
                y, e = quantise(x)
                j = torch.arange(x.shape[0], device=dev)
                p = self.table[s].long()[j // page]
                _bytes(c.values)[p, :, j % page] = _bytes(y)
                _bytes(c.scales)[p, :, j % page] = _bytes(e)
                rows[s] = held(y, e)
            caches.append(c)
        self.k, self.v = caches


LENS = [1, 0, 7, 8, 9, 16, 31, 32, 33, 127, 128, 129, 500, 1025]
HEADS = [(32, 8, 128, 16, "heads"), (8, 8, 64, 8, "tokens"), (6, 3, 80, 24, "heads"), (16, 2, 256, 64, "tokens"),
         (48, 1, 128, 128, "heads"), (15, 5, 64, 32, "tokens"), (12, 4, 96, 40, "heads"), (1, 1, 16, 16, "heads"),
         (4, 2, 144, 16, "tokens"), (4, 1, 48, 16, "tokens"), (2, 2, 112, 8, "heads")]


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("heads,kv,dim,page,layout", HEADS)
def test_decode(dev, dtype, heads, kv, dim, page, layout):
    _say(f"decode {dtype} {heads}/{kv} x {dim}, pages of {page}, {layout}")
    b = QBatch(dev, [1] * len(LENS), [x - 1 for x in LENS], heads, kv, dim, page, dtype, layout, seed=heads + dim, decode=True)
    lse = torch.empty(len(LENS), heads, device=dev)
    b.check(b.run(lse=lse), lse=lse)
    b.check(b.run(window=33), window=33)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("heads,kv,dim,page,layout", HEADS)
def test_chunks(dev, dtype, heads, kv, dim, page, layout):
    _say(f"chunks {dtype} {heads}/{kv} x {dim}, pages of {page}, {layout}")
    n = [1, 5, 0, 64, 33, 1, 130, 17, 2]
    cached = [100, 0, 3, 17, 0, 900, 70, -9, 63]          # one sequence with fewer tokens than rows
    b = QBatch(dev, n, cached, heads, kv, dim, page, dtype, layout, seed=heads + dim)
    lse = torch.empty(sum(n), heads, device=dev)
    b.check(b.run(lse=lse), lse=lse)
    b.check(b.run(window=50), window=50)
    b.check(b.run(max_q=130))
    b.check(b.run(window=1, max_q=1), window=1)           # a max_q that is too small costs time only


def test_many_sequences(dev):
    """More sequences than a wave's lanes hold at a time, and more parts than a list: decode rows, then a ragged step."""
    _say("many sequences")
    rng = np.random.default_rng(4)
    b = QBatch(dev, [1] * 700, rng.integers(-1, 60, 700).tolist(), 4, 2, 64, seed=1, decode=True)
    b.check(b.run())
    n = rng.integers(0, 9, 300)
    n[::50] = 40
    b = QBatch(dev, n.tolist(), rng.integers(0, 90, 300).tolist(), 8, 2, 64, seed=2)
    b.check(b.run())


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_long_contexts(dev, dtype):
    _say(f"long contexts {dtype}")
    b = QBatch(dev, [1], [20000], 8, 2, 128, 64, dtype, seed=7, decode=True)
    b.check(b.run())
    b = QBatch(dev, [3, 70], [9000, 4000], 8, 2, 128, 16, dtype, "tokens", seed=8)
    b.check(b.run())
    b = QBatch(dev, [40, 300], [9000, 2000], 8, 1, 64, 16, dtype, seed=9)
    b.check(b.run())


@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
def test_scales_of_scores(dev, scale):
    _say(f"scale {scale}")
    b = QBatch(dev, [20, 1, 40], [30, 200, 0], 8, 2, 64, seed=3, spread=0.3)
    b.check(b.run(scale=scale), scale=scale)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_small_and_large_rows(dev, dtype):
    """Rows from 2^-100 to 2^60: the scales reach the products and not only their sums."""
    _say(f"rows of all sizes {dtype}")
    for n, decode in (([1] * 6, True), ([50, 1, 33, 20, 9, 70], False)):
        b = QBatch(dev, n, [40, 100, 3, 0, 64, 200], 8, 2, 64, dtype=dtype, seed=3, decode=decode, spread=0.0)
        g = torch.Generator(device=dev).manual_seed(1)
        # values of sizes that differ by far, keys of one size: the scores stay ordinary
        for s, L in enumerate(b.len):
            e = torch.randint(-100, 60, (max(L, 0), b.kv), generator=g, device=dev)
            j = torch.arange(max(L, 0), device=dev)
            p = b.table[s].long()[j // b.page]
            code = _bytes(b.v.scales)[p, :, j % b.page].int() + e
            _bytes(b.v.scales)[p, :, j % b.page] = code.to(torch.uint8)
            b.rows[1][s] = b.rows[1][s] * torch.exp2(e.double())[..., None]
        b.check(b.run())


@pytest.mark.parametrize("dim", [64, 128, 80])
def test_queries_of_uneven_columns(dev, dim):
    """Query and key rows whose columns differ by up to 2^30 and 2^12: sums of products of all sizes."""
    _say(f"uneven columns, {dim}")
    b = QBatch(dev, [70, 40], [30, 200], 8, 2, dim, seed=dim, spread=0.0)
    g = torch.Generator(device=dev).manual_seed(2)
    down = torch.randint(-30, 1, (b.q.shape[0], 1, dim), generator=g, device=dev)
    down[:, :, 0] = 0
    up = torch.randint(-3, 4, (b.q.shape[0], 8, 1), generator=g, device=dev)
    b.q = (b.q.float() * torch.exp2((down + up).float())).to(BF16)
    b.check(b.run())


def test_queries_that_are_not_finite(dev):
    """They reach their own rows only."""
    _say("queries that are not finite")
    b = QBatch(dev, [40, 50], [30, 0], 8, 2, 64, seed=5)
    want = b.run()
    for bad in (math.nan, math.inf, -math.inf):
        b2 = b.q.clone()
        b2[7, 3, 11] = b2[60, 1, 40] = bad
        got = paged.paged_attention(b2, b.k, b.v, b.table, b.lens, b.cu)
        odd = torch.zeros(got.shape[:2], dtype=torch.bool, device=dev)
        odd[7, 3] = odd[60, 1] = True
        assert bool(got[odd].isnan().any()) and torch.equal(got[~odd], want[~odd])


def test_rows_of_no_sequence_and_out_in_place(dev):
    _say("padded step, out in place")
    b = QBatch(dev, [0, 33, 7], [5, 60, 300], 8, 2, 64, seed=2)
    pad = 9
    q = torch.cat([b.q, torch.full((pad, 8, 64), math.nan, dtype=BF16, device=dev)])
    lse = torch.empty(q.shape[0], 8, device=dev)
    out = paged.paged_attention(q, b.k, b.v, b.table, b.lens, b.cu, lse=lse)
    b.check(out[:-pad], lse=lse[:-pad])
    assert bool((out[-pad:] == 0).all()) and bool((lse[-pad:] == -math.inf).all())
    again = paged.paged_attention(q, b.k, b.v, b.table, b.lens, b.cu, out=q)
    assert again is q and torch.equal(q[:-pad], out[:-pad])


def test_plain_and_quantised_calls_share_a_workspace(dev):
    _say("one workspace")
    ws = torch.zeros(paged.workspace_bytes(BF16, 8, 2, 64, ragged=True), dtype=torch.uint8, device=dev)
    one = QBatch(dev, [70, 1, 40], [300, 2000, 0], 8, 2, 64, seed=2)
    two = Batch(dev, [70, 1, 40], [300, 2000, 0], 8, 2, 64, seed=2)
    for _ in range(2):
        one.check(one.run(workspace=ws))
        two.check(two.run(workspace=ws))


def test_captured(dev):
    """Append, attention and read in one graph, replayed beside eager calls on other streams."""
    _say("captured append, attention and read")
    g = torch.Generator(device=dev).manual_seed(6)
    H, HK, D, page, pages = 8, 2, 64, 16, 40
    n, cached = [40, 1, 3], [60, 200, 0]
    T = sum(n)
    lens = torch.tensor([a + b for a, b in zip(n, cached)], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 40, 41, 44], dtype=torch.int32, device=dev)
    table = torch.randperm(39, generator=g, device=dev).view(3, 13).to(torch.int32)
    cos_sin = paged.rope_table(256, D, device=dev)
    w = torch.randn(D, generator=g, device=dev).to(BF16)
    caches = paged.allocate_quantized_cache(pages, HK, page, D, dev)
    all_slots, _ = paged.cache_slots(table, lens, page, pages, torch.cat([cu.new_zeros(1), lens.cumsum(0).int()]), int(lens.sum()))
    k0 = torch.randn(all_slots.shape[0], HK, D, generator=g, device=dev).to(BF16)
    paged.append_kv_(None, k0, k0, *caches, all_slots)
    qkv = torch.randn(T, H + 2 * HK, D, generator=g, device=dev).to(BF16)

    def run():
        slots, pos = paged.cache_slots(table, lens, page, pages, cu, T)
        q = paged.append_kv_(*qkv.split([H, HK, HK], 1), *caches, slots, pos, cos_sin, q_norm=w, k_norm=w)
        return (paged.paged_attention(q, *caches, table, lens, cu), *paged.read_kv(*caches, slots))

    want = run()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = run()
    side = torch.cuda.Stream()
    for i in range(4):
        qkv.normal_(generator=g)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        side.synchronize()
        copies = [x.clone() for x in got]
        want = run()
        torch.cuda.synchronize()
        for a, b in zip(copies, want):
            assert torch.equal(a, b), i


def test_two_streams(dev):
    """Append and attention on two streams at once: each as on its own."""
    _say("two streams")
    cases = [QBatch(dev, [70, 1, 40, 9], [3000, 2000, 0, 900], 8, 2, 64, seed=s) for s in (1, 2)]
    want = [b.run() for b in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(6):
        for i, (b, st) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(st):
                n = b.len[0]
                slots, _ = paged.cache_slots(b.table[:1], b.lens[:1], b.page, b.k.values.shape[0],
                                             torch.tensor([0, n], dtype=torch.int32, device=dev), n)
                k, v = paged.read_kv(b.k, b.v, slots)
                paged.append_kv_(None, k, v, b.k, b.v, slots)            # the same rows again: their values do not change
                got[i].append(b.run())
    torch.cuda.synchronize()
    for x, y in zip(want, got):
        for z in y:
            assert torch.equal(x, z)


def test_registered_ops(dev):
    _say("registered ops")
    g = torch.Generator(device=dev).manual_seed(9)
    B, page, pages, n, H, HK, D = 3, 16, 24, [1, 9, 30], 8, 2, 64
    T = sum(n)
    lens = torch.tensor([50, 9, 100], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 1, 10, 40], dtype=torch.int32, device=dev)
    table = torch.randperm(pages, generator=g, device=dev).view(B, 8).to(torch.int32)
    slots, pos = paged.cache_slots(table, lens, page, pages, cu, T)
    q, k, v = torch.randn(T, H + 2 * HK, D, generator=g, device=dev).to(BF16).split([H, HK, HK], 1)
    rope, w = paged.rope_table(128, D, device=dev), torch.randn(D, generator=g, device=dev).to(BF16)
    one, two = ([make_cache(dev, pages, HK, page, D) for _ in range(2)] for _ in range(2))
    for c in (*one, *two):
        _bytes(c.values).fill_(0x31)
        _bytes(c.scales).fill_(120)
    flat = lambda c: (c[0].values, c[1].values, c[0].scales, c[1].scales)  # noqa: E731
    q1 = ops.op("append_kv_normed")(q, k, v, *flat(one), slots, pos, rope, False, w, w, 1e-5)
    q2 = paged.append_kv_(q, k, v, *two, slots, pos, rope, q_norm=w, k_norm=w)
    assert torch.equal(q1, q2) and all(torch.equal(_bytes(a), _bytes(b)) for a, b in zip(flat(one), flat(two)))
    o1 = ops.op("paged_attention_e4m3")(q1, *flat(one), table, lens, cu, None, 0, max(n))
    assert torch.equal(o1, paged.paged_attention(q2, *two, table, lens, cu, max_q=max(n)))
    for a, b in zip(ops.op("read_kv")(*flat(one), slots, FP32), paged.read_kv(*two, slots, FP32)):
        assert torch.equal(a, b)


# ---------------------------------------------------------------------------
# The decoder
# ---------------------------------------------------------------------------
def test_decoder_layer(dev):
    """A decoder's layer with normed heads over a quantised cache: prompts, then a mixed step, then decode rows.

    What the cache holds and what attention gives are compared with float64 from the layer's own
    projections and rows, so each check has the tolerance of its operator.
    """
    _say("decoder layer")
    g = torch.Generator(device=dev).manual_seed(3)
    HIDDEN, H, HK, D, MLP, page, pages = 256, 8, 2, 64, 512, 16, 64

    def lin(n_in, slices, fuse=False):
        base = torch.nn.Linear(n_in, sum(slices), bias=False).to(device=dev, dtype=BF16)
        base.weight.data = (torch.randn(sum(slices), n_in, generator=g, device=dev) / n_in ** 0.5).to(BF16)
        return vllm_layers.SwitchedLoRALinear(base, 1, 16, num_slices=len(slices),
                                              output_slices=slices if len(slices) > 1 else None, fuse_swiglu=fuse)

    norm = lambda n: (1 + 0.2 * torch.randn(n, generator=g, device=dev)).to(BF16)  # noqa: E731
    layer = decoder.SwitchedDecoderLayer(lin(HIDDEN, (H * D, HK * D, HK * D)), lin(H * D, (HIDDEN,)),
                                         lin(HIDDEN, (MLP, MLP), True), lin(MLP, (HIDDEN,)), norm(HIDDEN), norm(HIDDEN), H, HK,
                                         D, q_norm=norm(D), k_norm=norm(D))
    dec = decoder.SwitchedDecoder([layer], norm(HIDDEN), 1)
    dec.finalize([16])
    rope = paged.rope_table(512, D, device=dev)
    B = 4
    table = torch.randperm(pages, generator=g, device=dev)[: B * 12].view(B, 12).to(torch.int32)
    caches = [make_cache(dev, pages, HK, page, D) for _ in range(2)]
    seen = {}
    layer.qkv.register_forward_hook(lambda m, i, o: seen.update(qkv=o[0].clone()))
    layer.o_proj.register_forward_hook(lambda m, i, o: seen.update(o=i[0].clone()))
    lens = np.zeros(B, np.int64)
    for n, decode in (([37, 5, 130, 1], False), ([1, 1, 20, 0], False), ([1, 1, 1, 1], True)):
        T = sum(n)
        lens += n
        cu = None if decode else torch.tensor(np.concatenate([[0], np.cumsum(n)]), dtype=torch.int32, device=dev)
        dlens = torch.tensor(lens, dtype=torch.int32, device=dev)
        step = decoder.PagedStep(table, dlens, page, pages, rope, cu, T)
        dec.route(torch.randint(0, 2, (T,), generator=g, device=dev))
        out = dec(torch.randn(T, HIDDEN, generator=g, device=dev).to(BF16), step, [tuple(caches)])
        assert bool(out.isfinite().all())
        q, k, v = (t.unflatten(1, (-1, D)) for t in seen["qkv"].split([H * D, HK * D, HK * D], 1))
        at = (step.slots // page, slice(None), step.slots % page)
        row = lambda c: (_bytes(c.values)[at].view(E4M3), _bytes(c.scales)[at].view(E8M0))  # noqa: E731
        want, err = _turned(*_normed(k, layer.k_norm, layer.eps), rope, step.positions, False)
        _check_quantised(*row(caches[0]), want, err)
        y, s = quantise(v)
        assert torch.equal(row(caches[1])[0].float(), y.float()) and torch.equal(_bytes(row(caches[1])[1]), _bytes(s))
        # attention over what the cache holds, with the queries that an append of the same rows gives
        spare = [make_cache(dev, pages, HK, page, D) for _ in range(2)]
        b = QBatch.__new__(QBatch)
        b.q = paged.append_kv_(q, k, v, *spare, step.slots, step.positions, rope, q_norm=layer.q_norm, k_norm=layer.k_norm, eps=layer.eps)
        b.n, b.len, b.heads, b.kv, b.dim, b.dtype = n, lens.tolist(), H, HK, D, BF16
        b.rows = [[], []]
        for s in range(B):
            L = int(lens[s])
            slots, _ = paged.cache_slots(table[s:s + 1], dlens[s:s + 1], page, pages, torch.tensor([0, L], dtype=torch.int32, device=dev), L)
            for rows, x in zip(b.rows, paged.read_kv(*caches, slots, FP32)):
                rows.append(x)
        b.check(seen["o"].view(T, H, D))
