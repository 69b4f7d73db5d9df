"""GPU parity of the quantised paged cache at its edges: the ends of the range, keys next to a border between e4m3
values, scales with strides of their own, rows of values that are all tiny, how a ragged call's work is cut.

References and tolerances are those of test_gpu_quantized.py, whose helpers these tests use; what a test adds to them
stands beside it.
"""

from __future__ import annotations

import math

import pytest
import torch

from granite_switch_amd import _lib, paged
from test_gpu_quantized import BF16, E4M3, E8M0, FP32, QBatch, _bytes, _say, _turned, exponents, held, make_cache

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# Append and read
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [128, 33])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("turned", [False, True])
def test_the_largest_rows_stay_finite(dev, dtype, dim, turned):
    """A finite row reads back finite, within 2^-4, up to the type's largest value: 256 2^120 is no number of either type."""
    _say(f"the largest rows {dtype} {dim} turned={turned}")
    big = torch.finfo(dtype).max
    tops = [big, -big, 1.9375 * 2.0 ** 127, 1.875 * 2.0 ** 127, 1.75 * 2.0 ** 127, -1.90625 * 2.0 ** 127]
    rows = [torch.full((dim,), t, dtype=torch.float64) for t in tops]
    rows += [torch.linspace(-1, 1, dim, dtype=torch.float64) * abs(t) for t in tops]
    k = torch.stack(rows).to(dtype)[:, None].to(dev)
    assert bool(k.isfinite().all())
    T = k.shape[0]
    slots, caches = torch.arange(T, device=dev), [make_cache(dev, 2, 1, 16, dim) for _ in range(2)]
    # position 0 turns by nothing, through the keys' own arithmetic
    turn = (torch.zeros(T, dtype=torch.int64, device=dev), paged.rope_table(4, dim // 2 * 2, device=dev)) if turned else ()
    paged.append_kv_(None, k, -k, *caches, slots, *turn)
    for to in (BF16, FP32):
        for got, want in zip(paged.read_kv(*caches, slots, to), (k, -k)):
            off = (got.double() - want.double()).abs()
            assert int((~got.isfinite()).sum()) == 0
            assert bool((off <= want.double().abs() * 2.0 ** -4 + 2.0 ** 110).all())
    # beside a value that is not finite, too
    for bad in (math.nan, math.inf):
        odd = k.clone()
        odd[:, 0, 1] = bad
        paged.append_kv_(None, odd, odd, *caches, slots)
        got = paged.read_kv(*caches, slots)[0]
        assert bool(got[:, 0, 1].isnan().all())
        got[:, 0, 1] = 0
        assert int((~got.isfinite()).sum()) == 0


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("dim", [128, 33])
def test_read_of_every_scale(dev, dtype, dim):
    """Every scale byte times every value: x = y 2^e to the nearest, NaN for 255, an infinity where the type ends."""
    _say(f"read of every scale {dtype} {dim}")
    kc, vc = (make_cache(dev, 16, 1, 16, dim) for _ in range(2))
    for c, first in ((kc, 0), (vc, 128)):
        _bytes(c.scales).copy_(torch.arange(256, device=dev).view(16, 1, 16))
        _bytes(c.values).copy_((first + torch.arange(dim, device=dev) * 5) % 256)
    got = paged.read_kv(kc, vc, torch.arange(256, device=dev), dtype)
    for x, c in zip(got, (kc, vc)):
        want = held(c.values.transpose(1, 2).flatten(0, 1), c.scales.transpose(1, 2).flatten(0, 1))
        want[255] = math.nan
        least = 2.0 ** -126                                # below it the conversion may leave nothing
        x = x.double()
        assert torch.equal(x.isnan(), want.isnan())
        ends = want.abs() > torch.finfo(dtype).max
        assert bool((x[ends].abs() == math.inf).all()) and torch.equal(x[ends].sign(), want[ends].sign())
        exact = ~want.isnan() & ~ends & ((want.abs() >= least) | (want == 0))
        assert torch.equal(x[exact], want[exact])
        rest = ~want.isnan() & ~ends & ~exact
        assert bool((x[rest].abs() <= least).all())


def _rounded(y):
    """The e4m3 value nearest to float64 y (at most 448 + 16), ties to even, without a float32 between."""
    step = torch.exp2((torch.frexp(y)[1] - 1).clamp(min=-6).double() - 3)
    return torch.round(y / step) * step


def _exact_bytes(rows):
    """(values as float64, scale bytes) of float64 rows."""
    e = exponents(rows)
    return _rounded(rows * torch.exp2(-e.double())[..., None]), (e + 127).to(torch.uint8)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("turn", ["halves", "pairs", "norm only"])
def test_keys_are_rounded_from_64_bits(dev, dtype, turn):
    """Normed and rotated keys: the e4m3 values nearest to the exact ones, of 10^7 of which fp32 would move some ten.

    Exact where 64-bit arithmetic leaves no doubt: sums, a root and products of it are within 10^-13 of the row's largest
    value.
    """
    _say(f"keys from 64 bits {dtype} {turn}")
    g = torch.Generator(device=dev).manual_seed(11)
    T, HK, D, page = 10240, 8, 128, 64
    k = torch.randn(T, HK, D, generator=g, device=dev).to(dtype)
    w = (1 + 0.3 * torch.randn(D, generator=g, device=dev)).to(dtype)
    pos, table = torch.randint(0, 4000, (T,), generator=g, device=dev), paged.rope_table(4000, D, device=dev)
    caches, slots = [make_cache(dev, T // page, HK, page, D) for _ in range(2)], torch.arange(T, device=dev)
    rope = () if turn == "norm only" else (pos, table)
    paged.append_kv_(None, k, k, *caches, slots, *rope, interleaved=turn == "pairs", k_norm=w, eps=1e-5)
    x = k.double()
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + torch.tensor(1e-5).double()) * w.double()
    if rope:
        x = _turned(x, 0.0, table, pos, turn == "pairs")[0]
    values, scales = (_bytes(c).transpose(1, 2).flatten(0, 1) for c in caches[0])
    top = x.abs().amax(-1)
    sure = exponents((top * (1 + 1e-13))[..., None]) == exponents((top * (1 - 1e-13))[..., None])
    want, code = _exact_bytes(x)
    assert int((scales != code)[sure].sum()) == 0
    y = x * torch.exp2(127.0 - code.double())[..., None]
    firm = sure[..., None] & (_rounded(y + 448e-13) == _rounded(y - 448e-13))
    assert int((~firm).sum()) < 100
    moved = int((values.view(E4M3).double() != want)[firm].sum())
    assert moved == 0, moved


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_keys_next_to_a_border(dev, dtype):
    """Rotated keys 2^-30 from a midpoint between e4m3 values, and from 448: fp32 holds none of these apart from it."""
    _say(f"keys next to a border {dtype}")
    rows = torch.zeros(4, 1, 128, dtype=torch.float64)      # pairs (j, j + 64), turned to (p + q, q - p)
    p, q = rows[..., :64], rows[..., 64:]
    p[:, 0, :] = 1.0
    for r, tiny in enumerate((2.0 ** -30, -2.0 ** -30)):
        p[r, 0, :6], q[r, 0, :6] = torch.tensor([17.0, 19, 34, 2.125, 300, 136]), tiny
        p[2 + r, 0, :2], q[2 + r, 0, :2] = torch.tensor([448.0, 17]), tiny * 2 ** 5
    k = rows.to(dtype).to(dev)
    assert torch.equal(k.double().cpu(), rows)
    table = torch.cat([torch.ones(1, 64), -torch.ones(1, 64)], 1).to(dev)
    caches, slots = [make_cache(dev, 1, 1, 16, 128) for _ in range(2)], torch.arange(4, device=dev)
    paged.append_kv_(None, k, k, *caches, slots, torch.zeros(4, dtype=torch.int64, device=dev), table)
    want, code = _exact_bytes(torch.cat([p + q, q - p], -1).to(dev))
    assert code.flatten().tolist() == [127, 127, 128, 128]
    assert torch.equal(_bytes(caches[0].scales)[0, 0, :4], code.flatten())
    assert torch.equal(caches[0].values[0, 0, :4].double(), want[:, 0])


def test_scales_with_strides_of_their_own(dev):
    """Keys' and values' scales apart from each other's, in append, read and attention of both forms."""
    _say("strided scales")
    b = QBatch(dev, [1, 60, 3], [30, 300, 0], 8, 2, 64, seed=4)
    pages, kv, page = b.k.scales.shape
    out, one = b.run(), (b.k, b.v)
    big = [torch.full((pages + 1, kv + 1 + i, (2 + i) * page), 255, dtype=torch.uint8, device=dev) for i in range(2)]
    two = []
    for i, (c, x) in enumerate(zip(one, big)):
        scales = x[i:, 1:][:pages, :kv, i * page:(i + 1) * page]
        scales.copy_(_bytes(c.scales))
        two.append(paged.QuantizedCache(c.values, scales.view(E8M0)))
    assert two[0].scales.stride() != two[1].scales.stride()
    n = b.len[1]
    slots, _ = paged.cache_slots(b.table[1:2], b.lens[1:2], page, pages, torch.tensor([0, n], dtype=torch.int32, device=dev), n)
    for x, y in zip(paged.read_kv(*one, slots), paged.read_kv(*two, slots)):
        assert torch.equal(x, y)
    assert not torch.equal(*paged.read_kv(*one, slots))
    for kw in ({}, {"max_q": 60}):
        assert torch.equal(paged.paged_attention(b.q, *two, b.table, b.lens, b.cu, **kw), out)
    few = paged.paged_attention(b.q[:1], *one, b.table[:1], b.lens[:1])
    assert torch.equal(paged.paged_attention(b.q[:1], *two, b.table[:1], b.lens[:1]), few)
    k, v = (torch.randn(n, kv, 64, generator=torch.Generator(device=dev).manual_seed(i), device=dev).to(BF16) for i in (5, 6))
    for cache in (one, two):
        paged.append_kv_(None, k, 100 * v, *cache, slots)
    for c, x, keep in zip(one, two, big):
        assert torch.equal(_bytes(c.scales), _bytes(x.scales))
    for x in (*paged.read_kv(*two, slots),):
        assert int(x.isnan().sum()) == 0


# ---------------------------------------------------------------------------
# How a call's work is cut
# ---------------------------------------------------------------------------
def _row_parts(b, **kw):
    """Partial results of the row form that a call leaves for each key/value head, from its workspace."""
    ws = torch.zeros(paged.workspace_bytes(b.dtype, b.heads, b.kv, b.dim, ragged=True), dtype=torch.uint8, device=b.q.device)
    ws[_lib.GS_PAGED_HEAD_BYTES:] = 0xA5
    b.check(b.run(workspace=ws, **kw))
    cus = torch.cuda.get_device_properties(b.q.device).multi_processor_count
    rows, width = min(16, max(n for n in b.n if n * b.heads // b.kv <= 16) * b.heads // b.kv), 64 if b.dim <= 64 else 128
    most = (2 * 2 * cus + b.kv - 1) // b.kv + 1           # of a head
    left = ws[_lib.GS_PAGED_HEAD_BYTES:].view(torch.int32)[: b.kv * most * (16 * width + 32)]
    sums = left.view(b.kv, most, 16 * width + 32)[:, :, : rows * b.dim]
    found = (sums != -0x5A5A5A5B).any(-1).sum(1)
    assert int(found.min()) == int(found.max())
    return int(found[0])


@pytest.mark.parametrize("kv,n,cached", [(8, [3], [8189]), (8, [3, 1, 2], [4100, 9000, 16000]), (1, [5], [8187])])
def test_short_rows_without_chunks_fill_the_card(dev, kv, n, cached):
    """A batch that has row parts only is cut for the workgroups that there are, down to 4 units of 128 keys a part, also
    where the caller does not know max_q."""
    _say(f"row parts of a ragged call, {kv} heads, {n} over {cached}")
    b = QBatch(dev, n, cached, kv, kv, 128, seed=kv)
    known, unknown = _row_parts(b, max_q=max(n)), _row_parts(b)
    units = sum(-(-x // 128) for x in b.len)
    assert known > 8 and unknown >= min(known // 2, units // 4), (known, unknown)


def test_short_rows_beside_chunks(dev):
    """Beside chunk parts a row part has 8 units of 128 keys at least."""
    _say("row parts beside chunk parts")
    b = QBatch(dev, [3, 70], [8189, 500], 8, 8, 128, seed=1)
    assert 2 <= _row_parts(b) <= 8192 // (8 * 128)


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def _against_exact(b, out, rounding, of_result=0.0):
    """``out`` against float64, within ``rounding`` beside what fp32 sums leave, all relative to A = sum_j p_j |v_j|, and
    within ``of_result`` relative to the result.

    Scores of D products are off by ds <= (D + 4) u scale sum |q||k|, a probability so by a factor within 1 +- 2 ds twice
    over, sums of L terms by L u; bf16 subnormals by 2^-134 each.
    """
    G, t, scale = b.heads // b.kv, 0, b.dim ** -0.5
    for n, L, k, v in zip(b.n, b.len, *b.rows):
        if n and L > 0:
            q = b.q[t:t + n].double().unflatten(1, (b.kv, G)).permute(1, 0, 2, 3).reshape(b.kv, n * G, b.dim)
            k, v = k.double().transpose(0, 1).contiguous(), v.double().transpose(0, 1).contiguous()        # [kv, L, dim]
            kt = k.transpose(1, 2).contiguous()
            hide = torch.arange(L, device=q.device)[None] > (L - n + torch.arange(n, device=q.device)).repeat_interleave(G)[:, None]
            sc = (torch.bmm(q, kt) * scale).masked_fill(hide, -math.inf)
            ds = ((b.dim + 4) * 2.0 ** -24 * scale * torch.bmm(q.abs(), kt.abs())).masked_fill(hide, 0).amax(-1, keepdim=True)
            p = torch.softmax(sc, -1).nan_to_num(0.0)
            ref, A = torch.bmm(p, v), torch.bmm(p, v.abs())
            got = out[t:t + n].double().unflatten(1, (b.kv, G)).permute(1, 0, 2, 3).reshape(b.kv, n * G, b.dim)
            tol = (4 * ds + (L + 64) * 2.0 ** -24 + rounding) * A + of_result * ref.abs() + 2.0 ** -133
            worst = float(((got - ref).abs() / tol).nan_to_num(9e9).max())
            assert worst <= 1, (n, L)
        t += n


def _put_value_scales(b, codes):
    """Gives every value row of sequence s the scale bytes codes(s, number of tokens) [tokens, kv]."""
    for s, L in enumerate(b.len):
        j = torch.arange(max(L, 0), device=b.q.device)
        at = (b.table[s].long()[j // b.page], slice(None), j % b.page)
        code = codes(s, max(L, 0)).to(torch.uint8)
        _bytes(b.v.scales)[at] = code
        b.rows[1][s] = held(_bytes(b.v.values)[at].view(E4M3), code.view(E8M0))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("decode", [True, False])
def test_sequences_of_tiny_or_large_values(dev, dtype, dim, decode):
    """One power of two for all of a sequence's values, from the least that append writes; then some of each in one."""
    _say(f"tiny and large values {dtype} {dim} decode={decode}")
    n = [1] * 7 if decode else [5, 1, 33, 20, 9, 70, 2]
    b = QBatch(dev, n, [40, 100, 3, 0, 64, 200, 300], 4, 2, dim, dtype=dtype, seed=dim, decode=decode, spread=0.0)
    g = torch.Generator(device=dev).manual_seed(1)
    rounding = 2.0 ** -7 * 1.01 if dtype == BF16 else 0.0    # a probability's and the result's
    for code in (1, 2, 6, 40, 63, 64, 130, 220):
        _put_value_scales(b, lambda s, L: torch.full((L, b.kv), code, device=dev))
        _against_exact(b, b.run(), rounding)
    _put_value_scales(b, lambda s, L: torch.randint(1, 100, (L, b.kv), generator=g, device=dev))
    _against_exact(b, b.run(), rounding)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_row_form_rounds_its_result_only(dev, dim):
    """Probabilities enter the row form's products as two bf16 numbers: off by 2^-16 of themselves, not 2^-8."""
    _say(f"probabilities of the row form, {dim}")
    for n, decode in (([1] * 6, True), ([3, 1, 2, 4, 1, 2], False)):
        b = QBatch(dev, n, [40, 100, 3, 700, 64, 2000], 4, 2, dim, seed=dim, decode=decode)
        _against_exact(b, b.run(), 2.0 ** -16 * 1.01, 2.0 ** -8 * 1.01)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("decode", [True, False])
def test_the_least_scale_byte(dev, dtype, dim, decode):
    """Byte 0 is 2^-127, as in ``read_kv``: for a sequence's values, for some of them, and for its keys."""
    _say(f"scale byte 0 {dtype} {dim} decode={decode}")
    n = [1] * 5 if decode else [5, 1, 33, 20, 70]
    b = QBatch(dev, n, [40, 100, 3, 64, 200], 4, 2, dim, dtype=dtype, seed=dim, decode=decode, spread=0.0)
    g = torch.Generator(device=dev).manual_seed(1)
    rounding = 2.0 ** -7 * 1.01 if dtype == BF16 else 0.0
    _put_value_scales(b, lambda s, L: torch.zeros(L, b.kv, device=dev))
    _against_exact(b, b.run(), rounding)
    _put_value_scales(b, lambda s, L: 70 * torch.randint(0, 2, (L, b.kv), generator=g, device=dev))
    _against_exact(b, b.run(), rounding)
    # keys of 2^-127 times at most 448, queries past 2^100: scores of 0.0001 at most without the power of two
    for s, L in enumerate(b.len):
        j = torch.arange(L, device=dev)
        at = (b.table[s].long()[j // b.page], slice(None), j % b.page)
        _bytes(b.k.scales)[at] = 0
        b.rows[0][s] = held(_bytes(b.k.values)[at].view(E4M3), _bytes(b.k.scales)[at].view(E8M0))
    b.q = (b.q.float() * 2.0 ** 118).to(dtype)
    _against_exact(b, b.run(), rounding)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_scales_that_are_nan(dev, dtype):
    """Byte 255: the rows that see it are not finite, other sequences are as without it."""
    _say(f"scale byte 255 {dtype}")
    b = QBatch(dev, [3, 40, 1], [50, 30, 400], 4, 2, 64, dtype=dtype, seed=3)
    want = b.run()
    for c in (b.k, b.v):
        kept = _bytes(c.scales).clone()
        at = b.table[0].long()[0]
        _bytes(c.scales)[at, :, 5] = 255
        got = b.run()
        assert int(got[:3].isfinite().all(-1).sum()) == 0
        assert torch.equal(got[3:], want[3:])
        _bytes(c.scales).copy_(kept)
