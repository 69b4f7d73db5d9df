"""The paged append and attention kernels' accesses, replayed on the host.

``gs_check_paged_addresses`` and ``gs_check_append_addresses`` walk every part,
lane and block with the kernels' own address arithmetic; a violation is an
access outside its tensor, an output row or column taken other than once, or a
partial result that is joined other than once.  No kernel is launched.
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from granite_switch_amd import _lib

BF16, FP32 = _lib.GS_DTYPE_BF16, _lib.GS_DTYPE_FP32


def _p(a):
    return None if a is None else a.ctypes.data


def _check_attention(dtype, lens, cu, heads, kv, dim, page, window, layout, cus=256, seed=0, slack=2):
    rng = np.random.default_rng(seed)
    lens = np.asarray(lens, dtype=np.int32)
    B = len(lens)
    T = B if cu is None else int(cu[-1])
    need = [-(-max(int(x), 0) // page) for x in lens]
    pages = max(1, sum(need) + slack)
    max_pages = max([1] + need)
    table = rng.integers(-3, pages + 3, size=(B, max_pages)).astype(np.int32)      # unused entries may be anything
    ids = rng.permutation(pages)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = ids[at:at + n]
        at += n
    if layout == "heads":
        ps, hs, rs = kv * page * dim, page * dim, dim
    else:
        ps, hs, rs = kv * page * dim, dim, kv * dim
    cu = None if cu is None else np.asarray(cu, dtype=np.int32)
    msg, checked = ctypes.create_string_buffer(256), ctypes.c_int64()
    bad = _lib.load().gs_check_paged_addresses(dtype, heads * dim, dim, ps, hs, rs, ps, hs, rs, pages, page, _p(table),
                                               max_pages, max_pages, _p(lens), _p(cu), B, T, heads, kv, dim, window,
                                               heads * dim, dim, cus, msg, 256, ctypes.byref(checked))
    assert bad == 0, (bad, msg.value.decode() or _lib.last_error())
    assert checked.value > 0


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("lens,heads,kv,dim,page,window,layout", [
    ([1], 4, 1, 64, 8, 0, "heads"),
    ([0], 4, 4, 128, 16, 0, "heads"),
    ([0, 1, 7, 8, 9, 31, 32, 33, 127, 128, 129], 8, 2, 128, 16, 0, "tokens"),
    ([4000, 3, 0, 700], 6, 3, 80, 24, 0, "heads"),
    ([4000, 3, 0, 700], 32, 1, 96, 40, 100, "tokens"),
    ([5000], 16, 2, 256, 64, 0, "heads"),
    ([5000, 5000], 5, 5, 64, 256, 1, "heads"),
    ([333] * 300, 4, 2, 64, 16, 0, "heads"),
    ([17, 0] * 300, 2, 1, 64, 8, 9, "heads"),
])
def test_decode_addresses(dtype, lens, heads, kv, dim, page, window, layout):
    _check_attention(dtype, lens, None, heads, kv, dim, page, window, layout, cus=16)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("n,cached,heads,kv,dim,page,window", [
    ([1, 5, 0, 64], [100, 0, 3, 17], 8, 2, 128, 16, 0),
    ([33, 1, 200], [0, 900, 5], 6, 3, 80, 24, 0),
    ([33, 1, 200], [0, 900, 5], 4, 4, 64, 8, 50),
    ([7], [-3], 4, 2, 64, 16, 0),                       # fewer cached tokens than queries: rows that see nothing
    ([40], [60], 48, 1, 128, 32, 33),
])
def test_chunk_addresses(dtype, n, cached, heads, kv, dim, page, window):
    cu = np.concatenate([[0], np.cumsum(n)])
    lens = np.asarray(n) + np.asarray(cached)
    _check_attention(dtype, lens, cu, heads, kv, dim, page, window, "heads", cus=16)
    _check_attention(dtype, lens, cu, heads, kv, dim, page, window, "tokens", cus=64)


def test_random_batches():
    rng = np.random.default_rng(5)
    for seed in range(40):
        kv, G = int(rng.integers(1, 5)), int(rng.choice([1, 2, 3, 4, 8, 20]))
        B = int(rng.integers(1, 12))
        n = rng.integers(0, 30, size=B)
        lens = n + rng.integers(-4, 700, size=B)
        cu = np.concatenate([[0], np.cumsum(n)])
        if cu[-1] == 0:
            continue
        _check_attention(int(rng.choice([BF16, FP32])), lens, cu, kv * G, kv, int(rng.choice([64, 80, 128, 256])),
                         int(rng.choice([8, 16, 24, 64])), int(rng.choice([0, 0, 1, 20, 300])),
                         str(rng.choice(["heads", "tokens"])), cus=int(rng.choice([1, 16, 256])), seed=seed)


@pytest.mark.parametrize("dtype,vec,dim,rot", [
    (BF16, 1, 128, 128), (BF16, 1, 128, 32), (BF16, 1, 80, 0), (BF16, 1, 96, 64), (BF16, 1, 512, 512), (BF16, 0, 58, 10),
    (BF16, 0, 7, 0), (FP32, 1, 64, 32), (FP32, 1, 100, 8), (FP32, 0, 33, 32), (FP32, 0, 512, 512),
])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("tokens,heads,kv", [(1, 4, 1), (37, 0, 3), (300, 5, 2), (65, 40, 8)])
def test_append_addresses(dtype, vec, dim, rot, interleaved, tokens, heads, kv):
    rng = np.random.default_rng(tokens)
    page, pages, max_pos = 24, 20, 100
    slots = rng.integers(-2, pages * page + 2, size=tokens).astype(np.int64)
    pos = rng.integers(-1, max_pos + 1, size=tokens).astype(np.int64)
    msg, checked = ctypes.create_string_buffer(256), ctypes.c_int64()
    row = (heads + 2 * kv) * dim
    bad = _lib.load().gs_check_append_addresses(dtype, vec, row, dim, row, dim, tokens, heads, kv, dim, _p(pos), max_pos,
                                                rot, interleaved, _p(slots), kv * page * dim, page * dim, dim, pages,
                                                page, 64, msg, 256, ctypes.byref(checked))
    assert bad == 0, (bad, msg.value.decode() or _lib.last_error())
    assert checked.value > 0
