"""GPU parity of the paged cache: slots, rotated append, and attention.

References are plain float64 restatements, sequence by sequence.  Tolerances
follow from the arithmetic, with u = 2^-24 (fp32) and 2^-8 (bf16 rounding):

  append     a c - b s in fp32: 4 u (|a| + |b|), then one rounding to the type
  attention  a score of D products is off by at most ds = (D + 4) u scale sum |q||k|,
             so a probability by a factor within 1 +- 2 ds; sums of n terms by
             n u; bf16: each probability is rounded once (2^-8) and the result
             once more.  All of it relative to A = sum_j p_j |v_j|.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from granite_switch_amd import _lib, paged

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF16, FP32 = torch.bfloat16, torch.float32


def _say(msg):
    print(msg, flush=True)


# ---------------------------------------------------------------------------
# References
# ---------------------------------------------------------------------------
class Batch:
    """A ragged batch over a paged cache whose unused rows are NaN and whose unused table entries are junk."""

    def __init__(self, dev, n, cached, heads, kv, dim, page=16, dtype=BF16, layout="heads", seed=0, decode=False, pages=None):
        g = torch.Generator(device=dev).manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.n, self.len = list(n), [a + b for a, b in zip(n, cached)]
        self.heads, self.kv, self.dim, self.page, self.dtype = heads, kv, dim, page, dtype
        B, T = len(n), sum(n)
        need = [-(-max(L, 0) // page) for L in self.len]
        pages = pages or sum(need) + 3
        table = rng.integers(-5, pages + 5, size=(B, max(need + [1]) + 1))
        ids = rng.permutation(pages)[: sum(need)]
        if pages > 1000 and sum(need):
            ids[0] = pages - 1                             # the pool's last page is used
            ids[1:] = rng.permutation(pages - 1)[: sum(need) - 1]
        at = 0
        for s, m in enumerate(need):
            table[s, :m] = ids[at:at + m]
            at += m
        self.table = torch.tensor(table, dtype=torch.int32, device=dev)
        self.lens = torch.tensor(self.len, dtype=torch.int32, device=dev)
        self.cu = None if decode else torch.tensor(np.concatenate([[0], np.cumsum(n)]), dtype=torch.int32, device=dev)
        shape = (pages, kv, page, dim) if layout == "heads" else (pages, page, kv, dim)
        self.k, self.v = (torch.empty(shape, dtype=dtype, device=dev) for _ in range(2))
        self.rows = []
        for c in (self.k, self.v):
            if pages <= 4096:
                c.fill_(math.nan)
            if layout != "heads":
                c = c.permute(0, 2, 1, 3)
            rows = []
            for s, L in enumerate(self.len):
                x = torch.randn(max(L, 0), kv, dim, generator=g, device=dev).to(dtype)
                if L > 0:
                    j = torch.arange(L, device=dev)
                    p = self.table[s].long()[j // page]
                    if pages > 4096:
                        c[p.unique()] = math.nan
                    c[p, :, j % page] = x
                rows.append(x)
            self.rows.append(rows)
        if layout != "heads":
            self.k, self.v = self.k.permute(0, 2, 1, 3), self.v.permute(0, 2, 1, 3)
        self.q = (1.5 * torch.randn(T, heads, dim, generator=g, device=dev)).to(dtype)

    def run(self, window=0, scale=None, **kw):
        return paged.paged_attention(self.q, self.k, self.v, self.table, self.lens, self.cu, window=window, scale=scale, **kw)

    def check(self, out, window=0, scale=None, lse=None):
        scale = self.dim ** -0.5 if scale is None else scale
        G, t = self.heads // self.kv, 0
        for s, (n, L) in enumerate(zip(self.n, self.len)):
            for i0 in range(0, n, 128):
                m = min(128, n - i0)
                got = out[t + i0:t + i0 + m].double()
                k, v = (r[s].double() for r in self.rows)                                    # [L, kv, dim]
                q = self.q[t + i0:t + i0 + m].double().unflatten(1, (self.kv, G))
                p = L - n + i0 + torch.arange(m, device=out.device)
                j = torch.arange(max(L, 0), device=out.device)
                seen = j[None, :] <= p[:, None]
                if window:
                    seen &= j[None, :] > p[:, None] - window
                for h in range(self.kv):
                    qh, kh, vh = q[:, h].reshape(-1, self.dim), k[:, h].contiguous(), v[:, h].contiguous()
                    sc = (qh @ kh.T.contiguous()) * scale
                    ds = (self.dim + 4) * U * abs(scale) * (qh.abs() @ kh.abs().T.contiguous())
                    hide = ~seen.repeat_interleave(G, dim=0)
                    sc, ds = sc.masked_fill(hide, -math.inf), ds.masked_fill(hide, 0)
                    any_ = ~hide.all(dim=1) if L > 0 else torch.zeros(m * G, dtype=torch.bool, device=out.device)
                    pr = torch.softmax(sc, dim=1).nan_to_num(0.0) if L > 0 else sc
                    ref, A = pr @ vh, pr @ vh.abs()
                    dmax = ds.amax(dim=1, keepdim=True) if L > 0 else torch.zeros(m * G, 1, device=out.device).double()
                    rel = 4 * dmax + (max(L, 0) + 64) * U
                    if self.dtype == BF16:
                        rel = rel + 2.0 ** -7 * 1.01
                    tol = rel * A + 1e-30
                    g = got[:, h * G:(h + 1) * G].reshape(-1, self.dim)
                    err = (g - ref).abs()
                    assert not bool((~(err <= tol)).any()), (s, i0, h, float(err.max()), float((err / tol).nan_to_num(9e9).max()))
                    assert bool((g[~any_] == 0).all()), "a row that sees nothing is not zero"
                    if lse is not None:
                        want = torch.logsumexp(sc, dim=1) if L > 0 else torch.full((m * G,), -math.inf, device=out.device).double()
                        have = lse[t + i0:t + i0 + m, h * G:(h + 1) * G].reshape(-1).double()
                        assert bool((have[~any_] == -math.inf).all())
                        off = (have - want)[any_].abs()
                        ltol = (2 * dmax[:, 0] + (max(L, 0) + 64) * U + 8 * U * want.abs().nan_to_num(0.0, 0.0, 0.0))[any_]
                        assert bool((off <= ltol).all()), (s, float(off.max()))
            t += n


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
LENS = [1, 0, 7, 8, 9, 16, 31, 32, 33, 127, 128, 129, 500, 1025]


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("heads,kv,dim,page,layout", [
    (32, 8, 128, 16, "heads"), (8, 8, 64, 8, "tokens"), (6, 3, 80, 24, "heads"), (16, 2, 256, 64, "tokens"),
    (48, 1, 128, 128, "heads"), (15, 5, 64, 32, "tokens"), (12, 4, 96, 40, "heads"), (1, 1, 16, 16, "heads"),
])
def test_decode(dev, dtype, heads, kv, dim, page, layout):
    _say(f"decode {dtype} {heads}/{kv} x {dim}, pages of {page}, {layout}")
    b = Batch(dev, [1] * len(LENS), [x - 1 for x in LENS], heads, kv, dim, page, dtype, layout, seed=heads + dim, decode=True)
    lse = torch.empty(len(LENS), heads, device=dev)
    out = b.run(lse=lse)
    torch.cuda.synchronize()
    b.check(out, lse=lse)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("window", [1, 5, 64, 1000])
def test_decode_window(dev, dtype, window):
    _say(f"decode {dtype} window {window}")
    b = Batch(dev, [1] * len(LENS), [x - 1 for x in LENS], 8, 2, 64, 16, dtype, seed=window, decode=True)
    out = b.run(window=window)
    torch.cuda.synchronize()
    b.check(out, window=window)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("batch,length", [(1, 1), (1, 40000), (3, 9001), (300, 77), (700, 3)])
def test_decode_batch_shapes(dev, dtype, batch, length):
    """One long sequence over every part; more sequences than a workgroup has threads."""
    _say(f"decode {dtype} {batch} x {length}")
    b = Batch(dev, [1] * batch, [length - 1] * batch, 4, 2, 128, 16, dtype, seed=batch, decode=True)
    out = b.run()
    torch.cuda.synchronize()
    b.check(out)


def test_decode_scales_and_large_scores(dev):
    """Scores in the hundreds: the running maximum moves by more than an fp32 exponent between blocks."""
    b = Batch(dev, [1] * 6, [299, 10, 1023, 64, 0, 2000], 8, 2, 128, seed=3, decode=True, dtype=FP32)
    for scale in (4.0, 1e-3, 0.0, -1.0):
        _say(f"scale {scale}")
        out = b.run(scale=scale)
        torch.cuda.synchronize()
        b.check(out, scale=scale)


CHUNKS = ([1, 5, 0, 64, 3, 130], [100, 0, 3, 17, 1300, 250])


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("heads,kv,dim,page,layout,window", [
    (8, 2, 128, 16, "heads", 0), (8, 2, 128, 16, "tokens", 70), (4, 4, 64, 8, "heads", 0), (6, 3, 80, 24, "heads", 33),
    (16, 2, 256, 64, "tokens", 0), (24, 1, 128, 32, "heads", 0), (15, 5, 64, 16, "heads", 1), (12, 4, 96, 40, "tokens", 0),
])
def test_chunks(dev, dtype, heads, kv, dim, page, layout, window):
    _say(f"chunks {dtype} {heads}/{kv} x {dim}, pages of {page}, {layout}, window {window}")
    b = Batch(dev, *CHUNKS, heads, kv, dim, page, dtype, layout, seed=dim + window)
    lse = torch.empty(sum(CHUNKS[0]), heads, device=dev)
    out = b.run(window=window, lse=lse, max_q=130)
    torch.cuda.synchronize()
    b.check(out, window=window, lse=lse)
    again = b.run(window=window)                     # without the hint
    torch.cuda.synchronize()
    b.check(again, window=window)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_prompts_with_nothing_cached(dev, dtype):
    b = Batch(dev, [700, 1, 333, 64], [0, 0, 0, 0], 8, 2, 128, dtype=dtype, seed=8)
    _say(f"prompts {dtype}")
    out = b.run()
    torch.cuda.synchronize()
    b.check(out)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_rows_that_see_nothing(dev, dtype):
    """Fewer cached tokens than query rows: the first rows have no position, and give zeros."""
    _say(f"rows that see nothing {dtype}")
    b = Batch(dev, [40, 3, 20], [-25, -3, 5], 8, 2, 64, dtype=dtype, seed=9)
    lse = torch.empty(63, 8, device=dev)
    out = b.run(lse=lse)
    torch.cuda.synchronize()
    b.check(out, lse=lse)
    assert bool((out[:25] == 0).all()) and bool((out[40:43] == 0).all())


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("batch,most,window", [(2, 20000, 0), (40, 6000, 0), (256, 2000, 0), (300, 900, 0), (40, 6000, 700)])
def test_decode_uneven(dev, dtype, batch, most, window):
    """Lengths from none to many times the mean: parts of all sizes, some items cut, some whole."""
    _say(f"decode uneven {dtype} {batch} up to {most} window {window}")
    rng = np.random.default_rng(batch)
    lens = (most * rng.random(batch) ** 4).astype(int)
    lens[0] = most
    b = Batch(dev, [1] * batch, [x - 1 for x in lens.tolist()], 4, 2, 64, 16, dtype, seed=batch, decode=True)
    lse = torch.empty(batch, 4, device=dev)
    out = b.run(lse=lse, window=window)
    torch.cuda.synchronize()
    b.check(out, lse=lse, window=window)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_decode_many_short(dev, dtype):
    """70000 sequences of one token or none: more parts than 16-bit counts hold, lists of parts filled again and again."""
    _say(f"decode 70000 x 1 {dtype}")
    B, kv, dim, page = 70000, 1, 16, 8
    g = torch.Generator(device=dev).manual_seed(12)
    k, v = (torch.randn(B, kv, page, dim, generator=g, device=dev).to(dtype) for _ in range(2))
    q = torch.randn(B, 2, dim, generator=g, device=dev).to(dtype)
    table = torch.randperm(B, generator=g, device=dev).to(torch.int32)[:, None].contiguous()
    lens = torch.randint(0, 2, (B,), generator=g, device=dev).to(torch.int32)
    out = paged.paged_attention(q, k, v, table, lens)
    torch.cuda.synchronize()
    want = v[table[:, 0].long(), 0, 0] * lens[:, None].to(dtype)      # a softmax over one key is 1
    assert torch.equal(out, want[:, None].expand_as(out))


@pytest.mark.parametrize("heads,kv,dim,batch,most,window", [(8, 2, 128, 24, 7000, 0), (8, 2, 64, 24, 7000, 600),
                                                            (4, 4, 128, 330, 700, 0), (16, 1, 96, 12, 3000, 0)])
def test_ragged_uneven(dev, heads, kv, dim, batch, most, window):
    """Decode rows, short and long chunks in one batch, over caches of all lengths: both forms, tiles cut and whole."""
    _say(f"ragged uneven {heads}/{kv} x {dim} {batch} up to {most} window {window}")
    rng = np.random.default_rng(heads + batch)
    n = rng.choice([0, 1, 1, 2, 3, 4, 5, 17, 64, 129], size=batch).tolist()
    cached = (most * rng.random(batch) ** 4).astype(int)
    cached[-1] = most
    n[-1] = 40
    b = Batch(dev, n, cached.tolist(), heads, kv, dim, 16, BF16, seed=batch)
    lse = torch.empty(sum(n), heads, device=dev)
    out = b.run(window=window, lse=lse)
    torch.cuda.synchronize()
    b.check(out, window=window, lse=lse)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_large_pool(dev, dtype):
    """Element offsets past 2^32: the pool's last page is used."""
    dim, kv, page = 128, 2, 16
    pages = (1 << 32) // (kv * page * dim) + 77
    _say(f"pool of {pages} pages, {dtype}")
    b = Batch(dev, [1, 60], [300, 200], 8, kv, dim, page, dtype, seed=4, pages=pages)
    out = b.run()
    torch.cuda.synchronize()
    b.check(out)


def test_strided_queries_and_output(dev):
    """q as a slice of the QKV projection's rows, out into a wider buffer."""
    _say("strided q and out")
    b = Batch(dev, [1, 30, 5], [50, 10, 700], 8, 2, 128, seed=5)
    T = b.q.shape[0]
    qkv = torch.randn(T, 12 * 128, device=dev).to(BF16)
    qkv[:, :1024] = b.q.flatten(1)
    b.q = qkv[:, :1024].unflatten(1, (8, 128))
    buf = torch.full((T, 10, 128), 7.0, dtype=BF16, device=dev)
    out = b.run(out=buf[:, 1:9])
    torch.cuda.synchronize()
    b.check(out)
    assert bool((buf[:, 0] == 7).all()) and bool((buf[:, 9] == 7).all()), "columns outside out were written"


def test_streams_and_repeatability(dev):
    """Calls on two streams at once, each with its own workspace; the same bits every time."""
    _say("two streams")
    bs = [Batch(dev, [1] * 40, [1200 + 13 * i for i in range(40)], 8, 2, 128, seed=s, decode=True) for s in (1, 2)]
    want = [b.run() for b in bs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(bs[i].run())
    torch.cuda.synchronize()
    for i in range(2):
        bs[i].check(want[i])
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_graph_replays_follow_the_lengths(dev):
    """A decode step captured once and replayed as the sequences grow: append, then attention."""
    _say("graph")
    b = Batch(dev, [1] * 9, [0, 15, 16, 200, 1000, 3, 64, 127, 128], 8, 2, 128, seed=6, decode=True)
    b.table = torch.arange(9 * 70, device=dev, dtype=torch.int32).reshape(9, 70)
    b.k, b.v = (torch.randn(9 * 70, 2, 16, 128, device=dev).to(BF16) for _ in range(2))
    kn, vn = (torch.randn(9, 2, 128, device=dev).to(BF16) for _ in range(2))
    cs = paged.rope_table(2048, 128, device=dev)

    def step():
        slots, pos = paged.cache_slots(b.table, b.lens, 16, b.k.shape[0])
        q = paged.append_kv_(b.q, kn, vn, b.k, b.v, slots, pos, cs)
        return paged.paged_attention(q, b.k, b.v, b.table, b.lens)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for r in range(4):
        b.lens += 1
        b.q.normal_()
        kn.normal_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(got, want), f"replay {r}"


# ---------------------------------------------------------------------------
# Slots and append
# ---------------------------------------------------------------------------
def test_cache_slots(dev):
    rng = np.random.default_rng(0)
    n, L = [1, 0, 5, 70, 2], [10, 4, 5, 100, 1]
    table = rng.permutation(200)[:5 * 8].reshape(5, 8)
    table[2, 0] = -1
    cu = np.concatenate([[0], np.cumsum(n)])
    T = int(cu[-1]) + 3                                   # rows past the last sequence
    slots, pos = paged.cache_slots(torch.tensor(table, dtype=torch.int32, device=dev),
                                   torch.tensor(L, dtype=torch.int32, device=dev), 16, 200,
                                   torch.tensor(cu, dtype=torch.int32, device=dev), T)
    want_s, want_p = np.full(T, -1), np.zeros(T, dtype=np.int64)
    for s in range(5):
        for i in range(n[s]):
            p = L[s] - n[s] + i
            want_p[cu[s] + i] = max(p, 0)
            if p >= 0 and table[s, p // 16] >= 0:
                want_s[cu[s] + i] = table[s, p // 16] * 16 + p % 16
    assert np.array_equal(slots.cpu().numpy(), want_s) and np.array_equal(pos.cpu().numpy(), want_p)
    # one row per sequence; a length past the page table has no slot
    slots, pos = paged.cache_slots(torch.tensor(table[:, :2].copy(), dtype=torch.int32, device=dev),
                                   torch.tensor([1, 0, 33, 17, 32], dtype=torch.int32, device=dev), 16, 200)
    assert slots.tolist() == [table[0, 0] * 16, -1, -1, table[3, 1] * 16, table[4, 1] * 16 + 15]
    assert pos.tolist() == [0, 0, 32, 16, 31]


def _rotated(x, pos, cs, interleaved):
    """float64 rotation of x [T, heads, D], and |a| + |b| of each element's pair."""
    x = x.double()
    R = 0 if cs is None else cs.shape[1]
    out, mag = x.clone(), x.abs()
    if R:
        c, s = (t[:, None, :] for t in cs.double()[pos].chunk(2, dim=1))
        i0, i1 = (torch.arange(0, R, 2), torch.arange(1, R, 2)) if interleaved else (torch.arange(R // 2), torch.arange(R // 2, R))
        a, b = x[..., i0], x[..., i1]
        out[..., i0], out[..., i1] = a * c - b * s, b * c + a * s
        mag[..., i0] = mag[..., i1] = a.abs() + b.abs()
    return out, mag


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,heads,kv,dim,rot,page,layout", [
    (1, 32, 8, 128, 128, 16, "heads"), (300, 32, 8, 128, 128, 16, "tokens"), (37, 6, 3, 80, 32, 24, "heads"),
    (65, 12, 4, 96, 96, 8, "heads"), (19, 3, 1, 58, 10, 7, "tokens"), (5, 0, 2, 64, 64, 16, "heads"),
    (130, 16, 2, 256, 128, 64, "heads"), (4, 4, 4, 64, 0, 16, "heads"), (3, 2, 1, 5, 4, 1, "heads"),
])
def test_append(dev, dtype, interleaved, T, heads, kv, dim, rot, page, layout):
    _say(f"append {dtype} T={T} {heads}/{kv} x {dim} rot {rot} pages of {page} {layout} {'pairs' if interleaved else 'half'}")
    g = torch.Generator(device=dev).manual_seed(T + dim)
    qkv = torch.randn(T, (heads + 2 * kv) * dim, generator=g, device=dev).to(dtype)
    q, k, v = qkv.split([heads * dim, kv * dim, kv * dim], dim=1)
    q = q.unflatten(1, (heads, dim)) if heads else None
    k, v = k.unflatten(1, (kv, dim)), v.unflatten(1, (kv, dim))
    pages = T // page + 4
    shape = (pages, kv, page, dim) if layout == "heads" else (pages, page, kv, dim)
    kc, vc = (torch.randn(shape, generator=g, device=dev).to(dtype) for _ in range(2))
    if layout != "heads":
        kc, vc = kc.permute(0, 2, 1, 3), vc.permute(0, 2, 1, 3)
    slots = torch.randperm(pages * page, generator=g, device=dev)[:T]
    slots[torch.rand(T, generator=g, device=dev) < 0.15] = -1
    if T > 4:
        slots[2] = pages * page                        # past the pool: not stored
    cs = paged.rope_table(500, rot, device=dev) if rot else None
    pos = torch.randint(0, 500, (T,), generator=g, device=dev)
    kw, vw, mag_k = kc.double(), vc.double(), torch.zeros_like(kc, dtype=torch.float64)
    live = torch.nonzero((slots >= 0) & (slots < pages * page)).flatten()
    kr, mk = _rotated(k, pos, cs, interleaved)
    p, r = slots[live] // page, slots[live] % page
    kw[p, :, r], vw[p, :, r], mag_k[p, :, r] = kr[live], v.double()[live], mk[live]
    keep = qkv.clone()
    out = paged.append_kv_(q, k, v, kc, vc, slots, pos, cs, interleaved=interleaved)
    torch.cuda.synchronize()
    assert torch.equal(qkv, keep), "an input was written"
    half = 2.0 ** -8 if dtype == BF16 else 0.0
    assert torch.equal(vc.double(), vw), "the value cache differs"
    err = (kc.double() - kw).abs()
    assert bool((err <= half * kw.abs() + 4 * U * mag_k).logical_or(mag_k.eq(0) & err.eq(0)).all()), float(err.max())
    if heads:
        qr, mq = _rotated(q, pos, cs, interleaved)
        err = (out.double() - qr).abs()
        assert bool((err <= half * qr.abs() + 4 * U * mq).all()), float(err.max())
        inplace = qkv.clone()
        qi = inplace[:, :heads * dim].unflatten(1, (heads, dim))
        paged.append_kv_(qi, k, v, kc, vc, slots, pos, cs, q_out=qi, interleaved=interleaved)
        torch.cuda.synchronize()
        assert torch.equal(qi, out), "in place differs"
        assert torch.equal(inplace[:, heads * dim:], keep[:, heads * dim:])
    else:
        assert out is None


def test_append_positions_outside_the_table(dev):
    """Clamped to the table's first and last row: nothing past it is read."""
    k = torch.randn(3, 1, 64, device=dev)
    kc, vc = paged.allocate_cache(1, 1, 8, 64, FP32, dev)
    cs = paged.rope_table(10, 64, device=dev)
    paged.append_kv_(None, k, k, kc, vc, torch.arange(3, device=dev), torch.tensor([-7, 9, 1 << 40], device=dev), cs)
    torch.cuda.synchronize()
    want, mag = _rotated(k, torch.tensor([0, 9, 9], device=dev), cs, False)
    assert bool(((kc[0, 0, :3] - want[:, 0]).abs() <= 4 * U * mag[:, 0]).all())


def test_rope_table_matches_float64():
    t = paged.rope_table(5000, 64, theta=1e6, device="cpu")
    p = 4999 * 1e6 ** (-np.arange(0, 64, 2) / 64)
    assert np.abs(t[4999].numpy() - np.concatenate([np.cos(p), np.sin(p)])).max() <= 2.0 ** -24


# ---------------------------------------------------------------------------
# Refusals
# ---------------------------------------------------------------------------
def test_attention_refusals(dev):
    b = Batch(dev, [1, 1], [20, 3], 8, 2, 64, decode=True)
    call = lambda **kw: paged.paged_attention(**{**dict(q=b.q, k_cache=b.k, v_cache=b.v, page_table=b.table, kv_lens=b.lens), **kw})  # noqa: E731
    for bad, err in [
        (dict(q=b.q.half()), TypeError), (dict(q=b.q[0]), ValueError), (dict(q=b.q[:, :7]), ValueError),
        (dict(q=b.q.float()), ValueError), (dict(q=b.q[:1]), ValueError), (dict(k_cache=b.k[:, :1]), ValueError),
        (dict(kv_lens=b.lens.long()), ValueError), (dict(page_table=b.table.long()), ValueError),
        (dict(page_table=b.table[:1]), ValueError), (dict(window=-1), ValueError), (dict(kv_lens=b.lens.cpu()), ValueError),
        (dict(cu_seqlens=torch.zeros(2, dtype=torch.int32, device=dev)), ValueError), (dict(out=b.q[:, :4]), ValueError),
        (dict(lse=torch.empty(2, 8, device=dev, dtype=torch.float64)), ValueError),
        (dict(workspace=torch.empty(16, dtype=torch.uint8, device=dev)), _lib.GraniteSwitchError),
        (dict(workspace=torch.empty(16, dtype=torch.float32, device=dev)), ValueError),
        (dict(k_cache=b.k[..., :63], v_cache=b.v[..., :63], q=b.q[..., :63]), _lib.GraniteSwitchError),
        (dict(q=torch.empty(2 * 8 * 64 + 1, dtype=BF16, device=dev)[1:].view(2, 8, 64)), _lib.GraniteSwitchError),
        (dict(k_cache=b.k[:, :, :12], v_cache=b.v[:, :, :12]), _lib.GraniteSwitchError),       # pages of 12 rows
        (dict(q=torch.empty(2, 8, 264, dtype=BF16, device=dev), k_cache=torch.empty(2, 2, 8, 264, dtype=BF16, device=dev),
              v_cache=torch.empty(2, 2, 8, 264, dtype=BF16, device=dev)), _lib.GraniteSwitchError),
    ]:
        with pytest.raises(err):
            call(**bad)
    assert call(q=b.q[:0], page_table=b.table[:0], kv_lens=b.lens[:0]).shape == (0, 8, 64)


def test_append_refusals(dev):
    k = torch.randn(3, 2, 64, device=dev)
    q = torch.randn(3, 4, 64, device=dev)
    kc, vc = paged.allocate_cache(2, 2, 8, 64, FP32, dev)
    slots, pos, cs = torch.arange(3, device=dev), torch.arange(3, device=dev), paged.rope_table(9, 64, device=dev)
    call = lambda **kw: paged.append_kv_(**{**dict(q=q, k=k, v=k, k_cache=kc, v_cache=vc, slots=slots, positions=pos, cos_sin=cs), **kw})  # noqa: E731
    call()
    for bad, err in [
        (dict(k=k.half()), TypeError), (dict(v=k[:2]), ValueError), (dict(q=q[..., :32]), ValueError),
        (dict(q=q[:2]), ValueError), (dict(slots=slots.int()), ValueError), (dict(slots=slots[:2]), ValueError),
        (dict(positions=None), ValueError), (dict(positions=pos.int()), ValueError), (dict(cos_sin=cs.double()), ValueError),
        (dict(cos_sin=paged.rope_table(9, 66, device=dev)), ValueError), (dict(k_cache=kc[:, :1], v_cache=vc[:, :1]), ValueError),
        (dict(k_cache=kc.bfloat16()), ValueError), (dict(q=None, q_out=q), ValueError), (dict(q_out=q[:, :2]), ValueError),
        (dict(slots=slots.cpu()), ValueError), (dict(v_cache=vc[:1]), ValueError),
    ]:
        with pytest.raises(err):
            call(**bad)
    assert paged.append_kv_(q[:0], k[:0], k[:0], kc, vc, slots[:0]).shape == (0, 4, 64)
