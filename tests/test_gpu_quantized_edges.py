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
from test_gpu_quantized import BF16, E4M3, E8M0, FP32, QBatch, _bytes, _say, held, make_cache

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
