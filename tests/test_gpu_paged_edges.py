"""GPU parity of the paged attention where a call's arguments, not its sizes, are unusual.

References and tolerances are those of ``test_gpu_paged``.
"""

from __future__ import annotations

import math

import pytest
import torch

from granite_switch_amd import _lib, norms, ops, paged
from test_gpu_paged import BF16, FP32, Batch, _say

pytestmark = pytest.mark.gpu


# Chunks of more and of fewer than 16 rows, masked tails and diagonals; with 4100 cached tokens on
# few heads, tiles that are cut into parts.
SCALED = [("whole", [40, 1, 130, 3], [25, 70, 0, 300], 8, 2), ("cut", [40, 1, 130], [4100, 900, 3000], 4, 2)]


@pytest.mark.parametrize("scale", [4.0, 1e-3, 0.0, -1.0, -0.05])
@pytest.mark.parametrize("name,n,cached,heads,kv", SCALED, ids=[c[0] for c in SCALED])
@pytest.mark.parametrize("dim,window", [(128, 0), (64, 0), (80, 50)])
def test_ragged_scales(dev, scale, name, n, cached, heads, kv, dim, window):
    """A scale of zero weighs every key that a row sees alike; a negative one turns the order round."""
    _say(f"ragged scale {scale} {name} x {dim} window {window}")
    b = Batch(dev, n, cached, heads, kv, dim, seed=dim)
    lse = torch.empty(sum(n), heads, device=dev)
    out = b.run(scale=scale, window=window, lse=lse)
    torch.cuda.synchronize()
    b.check(out, scale=scale, window=window, lse=lse)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 40, 2 ** 30])
def test_wide_windows(dev, dtype, window):
    """A window wider than any cache is none, for rows without a position too."""
    _say(f"window {window} {dtype}")
    b = Batch(dev, [40, 3, 20, 1], [-25, -3, 5, 200], 8, 2, 64, dtype=dtype, seed=9)
    out = b.run(window=window)
    torch.cuda.synchronize()
    b.check(out)
    assert torch.equal(out, b.run())


@pytest.mark.parametrize("dtype,dim,max_q", [(BF16, 64, 0), (BF16, 128, 40), (BF16, 256, 0), (FP32, 80, 0), (BF16, 64, 2)])
@pytest.mark.parametrize("before,after", [(0, 3), (2, 0), (1, 700)])
def test_rows_of_no_sequence(dev, dtype, dim, max_q, before, after):
    """A step padded to a fixed number of rows: those of no sequence give zeros, whatever out held."""
    _say(f"rows of no sequence {dtype} x {dim}: {before}, {after}")
    n = [2, 1, 1] if max_q == 2 else [5, 1, 40]
    b = Batch(dev, n, [10, 20, 30], 8, 2, dim, dtype=dtype, seed=dim)
    T = b.q.shape[0]
    pad = lambda m: torch.randn(m, 8, dim, device=dev).to(dtype)
    q = torch.cat([pad(before), b.q, pad(after)])
    wide = torch.full((q.shape[0], 10, dim), math.nan, dtype=dtype, device=dev)
    out, lse = wide[:, 1:9], torch.full((q.shape[0], 8), math.nan, device=dev)
    paged.paged_attention(q, b.k, b.v, b.table, b.lens, b.cu + before, out=out, lse=lse, max_q=max_q or None)
    torch.cuda.synchronize()
    b.check(out[before:before + T], lse=lse[before:before + T])
    edge = [*range(before), *range(before + T, q.shape[0])]
    assert bool((out[edge] == 0).all()) and bool((lse[edge] == -math.inf).all())
    assert bool(wide[:, 0].isnan().all()) and bool(wide[:, 9].isnan().all()), "columns outside out were written"


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (BF16, 256), (FP32, 64)])
def test_no_sequences(dev, dtype, dim):
    _say(f"no sequences {dtype} x {dim}")
    b = Batch(dev, [5], [10], 8, 2, dim, dtype=dtype)
    out, lse = torch.full_like(b.q, math.nan), torch.full((5, 8), math.nan, device=dev)
    got = paged.paged_attention(b.q, b.k, b.v, b.table[:0], b.lens[:0], b.cu[:1], out=out, lse=lse)
    torch.cuda.synchronize()
    assert got is out and bool((out == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("ragged", [False, True])
def test_graphs_beside_eager_calls(dev, ragged):
    """Two graphs captured on a stream that has a workspace, replayed on two others while it works: the same bits."""
    _say(f"graphs beside eager calls, ragged {ragged}")
    n = [1, 40, 3, 130, 1] if ragged else [1] * 40
    bs = [Batch(dev, n, [2100 + 613 * i % 3000 for i in range(len(n))], 8, 2, 128, seed=s, decode=not ragged) for s in (1, 2, 3)]
    want = [b.run() for b in bs]
    torch.cuda.synchronize()
    for b, w in zip(bs, want):
        b.check(w)
    home, others, graphs, outs = torch.cuda.Stream(), [torch.cuda.Stream(), torch.cuda.Stream()], [], []
    with torch.cuda.stream(home):
        bs[2].run()
    torch.cuda.synchronize()
    for b in bs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=home):
            b.run()
            outs.append(b.run())                           # two calls of one capture
        graphs.append(g)
    for _ in range(4):
        for o in outs:
            o.fill_(math.nan)
        torch.cuda.synchronize()
        eager = []
        for _ in range(3):
            for g, s in zip(graphs, others):
                with torch.cuda.stream(s):
                    g.replay()
            with torch.cuda.stream(home):
                eager.append(bs[2].run())
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want)), "a graph's result differs"
        assert all(torch.equal(e, want[2]) for e in eager), "an eager result differs"


def test_capture_ids(dev):
    """Each capture has an id of its own, the same on every stream that it forks to; none outside of one."""
    s, fork, x, ids = torch.cuda.Stream(), torch.cuda.Stream(), torch.zeros(8, device=dev), []
    torch.cuda.synchronize()
    assert _lib.capture_id(s.cuda_stream) == 0
    for _ in range(3):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            x.add_(1)
            ids.append(_lib.capture_id(s.cuda_stream))
            fork.wait_stream(s)
            with torch.cuda.stream(fork):
                x.add_(1)
                assert _lib.capture_id(fork.cuda_stream) == ids[-1]
            s.wait_stream(fork)
        assert _lib.capture_id(s.cuda_stream) == 0 and _lib.capture_id(fork.cuda_stream) == 0
    assert len(set(ids)) == 3 and 0 not in ids


@pytest.mark.parametrize("n,max_q", [([1, 1, 0, 2, 1, 4], 4), ([1, 1, 0, 2, 1, 4], 2), ([5, 1, 40, 130], 1), ([5, 1, 40, 130], 3)])
@pytest.mark.parametrize("heads,kv,dim,window", [(8, 2, 128, 0), (4, 4, 64, 90), (6, 3, 80, 0)])
def test_few_rows_by_hint(dev, n, max_q, heads, kv, dim, window):
    """max_q keeps a batch of short rows off the chunk form; one that is too small costs time, no rows."""
    _say(f"rows {n}, max_q {max_q}, {heads}/{kv} x {dim} window {window}")
    b = Batch(dev, n, [700, 3, 50, 0, 64, 2100][: len(n)], heads, kv, dim, seed=dim)
    out, lse = torch.full_like(b.q, math.nan), torch.full((sum(n), heads), math.nan, device=dev)
    b.run(window=window, max_q=max_q, out=out, lse=lse)
    torch.cuda.synchronize()
    b.check(out, window=window, lse=lse)


def test_sizes_past_32_bits(dev):
    """What the library takes as 32 bits is not cut to them: a wider window is none, other sizes are refused."""
    _say("sizes past 32 bits")
    b = Batch(dev, [5, 1, 40], [10, 20, 30], 8, 2, 64)
    want = b.run()
    assert not torch.equal(b.run(window=5), want)
    for window in (2 ** 31, 2 ** 32 + 5, 2 ** 63 - 1, 2 ** 70):
        assert torch.equal(b.run(window=window), want), window
    assert torch.equal(b.run(max_q=2 ** 32 + 1), want)
    for kw in (dict(page_size=2 ** 32 + 16), dict(page_size=-(2 ** 32) + 16)):
        with pytest.raises(ValueError, match="page_size"):
            paged.cache_slots(b.table, b.lens, num_pages=b.k.shape[0], cu_seqlens=b.cu, num_tokens=46, **kw)
    rows = torch.empty(1, 1, 1, 64, dtype=BF16, device=dev).expand(1, 1, 2 ** 32 + 16, 64)
    one, slots = torch.empty(1, 1, 64, dtype=BF16, device=dev), torch.zeros(1, dtype=torch.int64, device=dev)
    with pytest.raises(ValueError, match="rows"):
        paged.append_kv_(None, one, one, rows, rows, slots)
    with pytest.raises(ValueError, match="rows"):
        paged.paged_attention(one, rows, rows, b.table[:1], b.lens[:1])
    row = torch.empty(2 ** 32 + 8, dtype=BF16, device=dev)
    with pytest.raises(ValueError, match="hidden"):
        norms.residual_norm(row[None], row[None], row)


def test_registered_ops_and_autograd(dev):
    """The registered ops take tracked inputs as any op without a formula does: forward works, backward says so."""
    _say("registered ops, tracked inputs")
    b = Batch(dev, [5, 1, 40], [10, 20, 30], 8, 2, 64)
    want = b.run()
    q = b.q.clone().requires_grad_()
    got = ops.op("paged_attention")(q, b.k, b.v, b.table, b.lens, b.cu, None, 0, None)
    assert torch.equal(got, want)
    x, w = torch.randn(4, 64, device=dev, requires_grad=True), torch.ones(64, device=dev)
    y, r = ops.op("residual_norm")(x, torch.zeros(4, 64, device=dev), w, 1e-5, 1.0, None, None, None)
    assert torch.equal(r, x)
    k = torch.randn(3, 2, 64, device=dev).to(BF16).requires_grad_()
    slots = torch.arange(3, device=dev)
    ops.op("append_kv")(b.q[:3], k, k, b.k, b.v, slots, None, None, False)
    assert torch.equal(b.k[0, :, :3].transpose(0, 1), k)
    with pytest.raises(RuntimeError):
        got.sum().backward()


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_own_workspace(dev, dtype):
    """One workspace for calls of all kinds, one after the other: each leaves its counters at zero."""
    _say(f"own workspace {dtype}")
    n = [1, 40, 3, 130, 1]
    cached = [2100, 900, 5000, 3000, 0]
    ragged = Batch(dev, n, cached, 8, 2, 128, dtype=dtype, seed=1)
    decode = Batch(dev, [1] * 5, cached, 8, 2, 128, dtype=dtype, seed=2, decode=True)
    need = paged.workspace_bytes(dtype, 8, 2, 128, ragged=True)
    assert need >= paged.workspace_bytes(dtype, 8, 2, 128)
    ws = torch.full((need,), 255, dtype=torch.uint8, device=dev)
    ws[:_lib.GS_PAGED_HEAD_BYTES] = 0
    for b in (ragged, decode, ragged, decode):
        out = b.run(workspace=ws)
        torch.cuda.synchronize()
        assert not ws[:_lib.GS_PAGED_HEAD_BYTES].any()
        b.check(out)
        assert torch.equal(out, b.run())


@pytest.mark.parametrize("dtype,heads,kv,dim", [(BF16, 8, 2, 128), (BF16, 6, 2, 80), (BF16, 16, 2, 256), (FP32, 6, 2, 64)])
def test_out_in_place(dev, dtype, heads, kv, dim):
    """The result may take the queries' place."""
    _say(f"out is q {dtype} {heads}/{kv} x {dim}")
    for decode in (False, True):
        n = [1] * 4 if decode else [1, 40, 3, 130]
        b = Batch(dev, n, [4100, 900, 5000, 3000], heads, kv, dim, dtype=dtype, seed=3, decode=decode)
        want, q = b.run(), b.q.clone()
        got = paged.paged_attention(q, b.k, b.v, b.table, b.lens, b.cu, out=q)
        torch.cuda.synchronize()
        assert got is q and torch.equal(q, want)
