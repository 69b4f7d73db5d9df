"""Operators of a quantised paged cache and of normed heads, as cases that can be timed and compared.

  append   ``paged.append_kv_`` into a quantised cache, with the norms of queries
           and keys for each head: norm and rotation of q and k, k and v stored as
           e4m3 values with one power of two for each row; q returned
  read     ``paged.read_kv``: rows of a quantised cache, by their slots
  decode   ``paged.paged_attention`` over a quantised cache, one new token per
           sequence
  chunk    the same with ``cu_seqlens``: ragged query chunks (prompts, invocation
           tokens over a cached prefix, mixed steps)

A row of a quantised cache is a head's key or value of one token: values y in
e4m3 and the exponent e of a power of two, x = y 2^e, with e the least integer
that keeps the row's largest magnitude within 448 2^e (-126 at least).

Sizes are those of the benchmark and test configurations (32 query and 8
key/value heads of 128, 8 of 64; 256 decode requests at positions 16..2048,
8192-token prefills, the mixed step of 48 decode rows and 16 chunks of 256) or
generic ones.

Where ``own`` is false the operators run in their plain form: elementary torch
operations in 32 bits over a padded batch, rounded once at the end.
"""

from __future__ import annotations

import functools
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------
def _append(tokens, *, heads=32, kv=8, dim=128, rot=0, page=16, style="half", layout="heads", norm=True, quant=True,
            dtype="bf16", name=None):
    c = {"op": "append", "tokens": tokens, "heads": heads, "kv": kv, "dim": dim, "rot": rot or dim, "page": page,
         "style": style, "layout": layout, "norm": norm, "quant": quant, "dtype": dtype}
    return {"name": name, **c} if name else c


def _read(tokens, *, kv=8, dim=128, page=16, layout="heads", dtype="bf16", name=None):
    c = {"op": "read", "tokens": tokens, "kv": kv, "dim": dim, "page": page, "layout": layout, "dtype": dtype}
    return {"name": name, **c} if name else c


def _attn(op, *, decode=0, chunks=0, lo=1, hi=1, q_lo=1, q_hi=1, empty=0, total=0, heads=32, kv=8, dim=128, page=16,
          window=0, layout="heads", dtype="bf16", name=None):
    """``decode`` rows of one query and ``chunks`` sequences of q_lo..q_hi queries (``total``: scaled to this sum), each
    with lo..hi tokens cached before them; ``empty`` rows of a padded batch have nothing cached."""
    c = {"op": op, "decode": decode, "chunks": chunks, "lo": lo, "hi": hi, "q_lo": q_lo, "q_hi": q_hi, "empty": empty,
         "total": total, "heads": heads, "kv": kv, "dim": dim, "page": page, "window": window, "layout": layout,
         "dtype": dtype}
    return {"name": name, **c} if name else c


def listed():
    return [
        # a full decode batch: one row per request, each into its own page of a quantised cache
        _append(256, name="append_decode_t256"),
        # a large chunked prefill into a quantised cache: the most rows that one call stores
        _append(8192, page=64, name="append_prefill_t8192"),
        # the mixed step of a model with normed heads whose cache is not quantised
        _append(4144, quant=False, name="append_norm_t4144"),
        # fp32 evaluation of a small model without norms, rotary over half of each head, pairs side by side, an odd count
        _append(513, dim=64, rot=32, page=24, style="pairs", norm=False, dtype="fp32", name="append_fp32_d64_t513"),
        # a short conversation's cache read back, to be moved or looked at (latency only)
        _read(257, name="read_t257"),
        # a long document's cache read back: the most rows that one call reads
        _read(131071, page=64, name="read_t131071"),
        # a full decode batch, contexts as the decode workload has them
        _attn("decode", decode=256, lo=16, hi=2047, name="decode_b256"),
        # one conversation over a long document: the cache's length is all there is to split over
        _attn("decode", decode=1, lo=131071, hi=131071, page=64, name="decode_long_b1"),
        # fp32 evaluation, 64-wide heads, a sliding window, an odd batch
        _attn("decode", decode=19, lo=16, hi=8191, dim=64, window=1000, page=32, dtype="fp32", name="decode_fp32_window"),
        # adapters switched on mid-conversation: a few invocation tokens each over long cached prefixes
        _attn("chunk", chunks=8, lo=2048, hi=16384, q_lo=3, q_hi=64, name="chunk_invocation"),
        # a serving step: 48 decode rows and 16 prefill chunks of 256 with cached prefixes
        _attn("chunk", decode=48, chunks=16, lo=16, hi=3839, q_lo=256, q_hi=256, name="chunk_step_t4144"),
        # a large prefill: 16 prompts, log-uniform lengths, nothing cached before (the most arithmetic)
        _attn("chunk", chunks=16, lo=0, hi=0, q_lo=64, q_hi=2048, total=8192, page=64, name="chunk_prefill_t8192"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


# query heads, key/value heads, head width
HEADS = ((32, 8, 128), (32, 8, 128), (32, 8, 64), (40, 8, 64), (16, 16, 128), (8, 1, 128), (48, 1, 128), (12, 4, 96),
         (16, 2, 256), (6, 3, 80), (15, 5, 64))
PAGES = (16, 16, 32, 64, 128, 8, 24, 256)


def draw(rng):
    op = rng.choice(["append", "append", "read", "decode", "decode", "chunk", "chunk"])
    while True:
        heads, kv, dim = rng.choice(HEADS)
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        page = rng.choice(PAGES)
        layout = rng.choice(["heads", "heads", "tokens"])
        window = _log_int(rng, 16, 4096) if rng.random() < 0.25 else 0
        shape = dict(kv=kv, dim=dim, page=page, layout=layout, dtype=dtype)
        if op == "append":
            quant = rng.random() < 0.75
            case = _append(_log_int(rng, 1, 8192), heads=heads, rot=rng.choice([dim, dim, dim // 2, 16]),
                           style=rng.choice(["half", "half", "pairs"]), norm=not quant or rng.random() < 0.6, quant=quant,
                           **shape)
        elif op == "read":
            case = _read(_log_int(rng, 1, 131072), **shape)
        elif op == "decode":
            lo = _log_int(rng, 1, 4096)
            case = _attn("decode", decode=_log_int(rng, 1, 512), lo=lo, hi=_log_int(rng, lo, 131072), window=window,
                         empty=rng.choice([0, 0, 1, 3]), heads=heads, **shape)
        else:
            lo = rng.choice([0, _log_int(rng, 1, 8192)])
            q_lo = _log_int(rng, 1, 512)
            case = _attn("chunk", decode=rng.choice([0, 0, _log_int(rng, 1, 64)]), chunks=_log_int(rng, 1, 32), lo=lo,
                         hi=_log_int(rng, max(lo, 1), 16384) if lo else 0, q_lo=q_lo, q_hi=_log_int(rng, q_lo, 4096),
                         window=window, heads=heads, **shape)
        w = work(case)
        if w["bytes"] <= 8.0e8 and w["flops"] <= 5.0e10 and _padded(case) <= 2.0e9:
            return case


def _padded(case):
    """Elements of the largest tensor of the plain form (scores, or gathered keys)."""
    if case["op"] not in ("decode", "chunk"):
        return 0
    n, length = _lengths(case)
    return len(n) * max(length) * max(case["heads"] * max(n), case["kv"] * case["dim"])


def _lengths(case):
    return _lengths_of(tuple(case[k] for k in ("decode", "chunks", "lo", "hi", "q_lo", "q_hi", "empty", "total")))


@functools.lru_cache(maxsize=64)
def _lengths_of(key):
    """(queries, cached tokens with the queries among them) of each sequence; the same for every seed."""
    decode, chunks, lo, hi, q_lo, q_hi, empty, total = key
    rng = np.random.default_rng(list(key))

    def log_uniform(a, b, n):
        if b <= a:
            return np.full(n, a, dtype=np.int64)
        return np.clip(np.exp(rng.uniform(math.log(max(a, 1)), math.log(b + 1), size=n)).astype(np.int64), a, b)

    q = log_uniform(q_lo, q_hi, chunks)
    if total:
        q = np.maximum(1, q * total // q.sum())
        q[np.argmax(q)] += total - q.sum()
    n = np.concatenate([np.ones(decode, dtype=np.int64), q])
    length = log_uniform(lo, hi, decode + chunks) + n
    order = rng.permutation(len(n) + empty)
    n, length = np.concatenate([n, np.ones(empty, dtype=np.int64)]), np.concatenate([length, np.zeros(empty, dtype=np.int64)])
    return n[order].tolist(), length[order].tolist()


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _quantised(x):
    """(e4m3 values, e8m0 scales) of the rows of x, fp32."""
    m, e = torch.frexp(x.abs().amax(dim=-1))                     # m 2^e with m in [0.5, 1); 448 = 0.875 2^9
    e = torch.where(m > 0, torch.where(m <= 0.875, e - 9, e - 8), -126).clamp_(min=-126)
    return torch.ldexp(x, -e[..., None]).to(E4M3), (e + 127).to(torch.uint8).view(E8M0)


def _pool(case, pages, g, device):
    """A quantised cache: values [pages, kv, page, dim], a head's rows of a page side by side or a token's heads, and
    scales [pages, kv, page].  Rows differ in size, as a model's do."""
    kv, page, dim = case["kv"], case["page"], case["dim"]
    values = torch.empty((pages, kv, page, dim), dtype=E4M3, device=device)
    scales = torch.empty((pages, kv, page), dtype=torch.uint8, device=device).view(E8M0)
    step = max(1, (1 << 25) // (kv * page * dim))
    for at in range(0, pages, step):
        n = min(step, pages - at)
        x = torch.randn(n, kv, page, dim, generator=g, device=device)
        x *= torch.exp(0.5 * torch.randn(n, kv, page, 1, generator=g, device=device))
        y, s = _quantised(x)
        values[at:at + n].view(torch.uint8).copy_(y.view(torch.uint8))
        scales[at:at + n].view(torch.uint8).copy_(s.view(torch.uint8))
    if case["layout"] == "tokens":
        values = values.view(torch.uint8).permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3).view(E4M3)
    return values, scales


def _plain_pool(case, pages, g, device):
    """A cache that is not quantised, of the case's type."""
    kv, page, dim = case["kv"], case["page"], case["dim"]
    shape = (pages, kv, page, dim) if case["layout"] == "heads" else (pages, page, kv, dim)
    out = torch.randn(shape, generator=g, device=device).to(DTYPES[case["dtype"]])
    return out if case["layout"] == "heads" else out.permute(0, 2, 1, 3)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    normal = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    st = {"case": dict(case)}
    kv, dim, page = case["kv"], case["dim"], case["page"]
    if case["op"] in ("append", "read"):
        T = case["tokens"]
        # runs of slots in pages of random order, one slot in 50 a padding row (-1)
        pages = -(-T // page) + 3
        table = torch.randperm(pages, generator=g, device=dev)
        t = torch.arange(T, device=dev)
        slots = table[t // page] * page + t % page
        st["slots"] = torch.where(torch.rand(T, generator=g, device=dev) < 0.02, -1, slots)
        make = _pool if case.get("quant", True) else _plain_pool
        st["k_cache"], st["v_cache"] = make(case, pages, g, dev), make(case, pages, g, dev)
        if case["op"] == "read":
            return st
        H, R = case["heads"], case["rot"]
        # the QKV projection's output rows; q, k and v are views into them
        qkv = (normal(T, (H + 2 * kv) * dim) * torch.exp(0.5 * normal(T, 1))).to(dt)
        st["q"] = qkv[:, : H * dim].unflatten(1, (H, dim))
        st["k"] = qkv[:, H * dim: (H + kv) * dim].unflatten(1, (kv, dim))
        st["v"] = qkv[:, (H + kv) * dim:].unflatten(1, (kv, dim))
        st["q_norm"], st["k_norm"] = ((1 + 0.2 * normal(dim)).to(dt) for _ in range(2)) if case["norm"] else (None, None)
        most = 4096
        st["positions"] = torch.randint(0, most, (T,), generator=g, device=dev)
        inv = 10000.0 ** (-torch.arange(0, R, 2, device=dev, dtype=torch.float64) / R)
        ang = torch.arange(most, device=dev, dtype=torch.float64)[:, None] * inv[None, :]
        st["cos_sin"] = torch.cat([ang.cos(), ang.sin()], dim=1).float()
        return st
    n, length = _lengths(case)
    st["q"] = (2 * normal(sum(n), case["heads"], dim)).to(dt)
    need = [-(-x // page) for x in length]
    pages = sum(need) + 5
    st["k_cache"], st["v_cache"] = _pool(case, pages, g, dev), _pool(case, pages, g, dev)
    ids = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    at = torch.tensor([0] + np.cumsum(need)[:-1].tolist(), device=dev)
    cols = torch.arange(max(1, max(need)), device=dev)
    used = cols[None, :] < torch.tensor(need, device=dev)[:, None]
    st["page_table"] = torch.where(used, ids[(at[:, None] + cols[None, :]).clamp(max=pages - 1)], 0).contiguous()
    st["kv_lens"] = torch.tensor(length, dtype=torch.int32, device=dev)
    st["cu_seqlens"] = None
    if case["op"] == "chunk":
        st["cu_seqlens"] = torch.tensor([0] + np.cumsum(n).tolist(), dtype=torch.int32, device=dev)
    st["max_q"], st["max_kv"] = max(n), max(length)          # a scheduler has both on the host
    st["scale"] = dim ** -0.5
    return st


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(st):
    if own:
        return _run_own(st)
    op = st["case"]["op"]
    return _plain_append(st) if op == "append" else _plain_read(st) if op == "read" else _plain_attention(st)


def _run_own(st):
    from __graft_entry__ import load_package

    load_package()
    from granite_switch_amd import paged

    c = st["case"]
    k_cache, v_cache = st["k_cache"], st["v_cache"]
    if c.get("quant", True):
        k_cache, v_cache = paged.QuantizedCache(*k_cache), paged.QuantizedCache(*v_cache)
    if c["op"] == "append":
        q = paged.append_kv_(st["q"], st["k"], st["v"], k_cache, v_cache, st["slots"], positions=st["positions"],
                             cos_sin=st["cos_sin"], interleaved=c["style"] == "pairs", q_norm=st["q_norm"],
                             k_norm=st["k_norm"], eps=EPS)
        return q, st["k_cache"], st["v_cache"]
    if c["op"] == "read":
        return paged.read_kv(k_cache, v_cache, st["slots"], dtype=DTYPES[c["dtype"]])
    return paged.paged_attention(st["q"], k_cache, v_cache, st["page_table"], st["kv_lens"], cu_seqlens=st["cu_seqlens"],
                                 scale=st["scale"], window=c["window"], max_q=st["max_q"])


def _plain_append(st):
    c = st["case"]
    R, page = c["rot"], c["page"]
    cos, sin = st["cos_sin"][st["positions"]][:, None, :].chunk(2, dim=-1)

    def rotated(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * w.float()
        turn, rest = x[..., :R], x[..., R:]
        if c["style"] == "half":
            a, b = turn[..., : R // 2], turn[..., R // 2:]
            return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], dim=-1)
        a, b = turn[..., 0::2], turn[..., 1::2]
        return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2), rest], dim=-1)

    slots = st["slots"]
    kept = slots >= 0
    at = torch.where(kept, slots, 0)
    first, src0 = (slots == 0).any(), torch.argmax((slots == 0).to(torch.int32))

    def store(cache, rows):
        # a padding row stores nothing: it writes what the pool's first row will hold anyway
        mask = kept.view(-1, *[1] * (rows.dim() - 1))
        cache[at // page, :, at % page] = torch.where(mask, rows, torch.where(first, rows[src0], cache[0, :, 0]))

    for rows, cache in ((rotated(st["k"], st["k_norm"]), st["k_cache"]), (st["v"].float(), st["v_cache"])):
        if c["quant"]:
            for held, x in zip(cache, _quantised(rows)):
                store(held.view(torch.uint8), x.view(torch.uint8))
        else:
            store(cache, rows.to(cache.dtype))
    return rotated(st["q"], st["q_norm"]).to(st["q"].dtype), st["k_cache"], st["v_cache"]


def _dequantised(values, scales, index):
    """Rows ``index`` of the first dimension, fp32."""
    y = values.view(torch.uint8)[index].view(E4M3).float()
    return torch.ldexp(y, scales.view(torch.uint8)[index].to(torch.int32)[..., None] - 127)


def _plain_read(st):
    c, slots = st["case"], st["slots"]
    page = c["page"]
    at = slots.clamp(min=0)

    def rows(cache):
        values, scales = (t.view(torch.uint8)[at // page, :, at % page] for t in cache)
        x = torch.ldexp(values.view(E4M3).float(), scales.to(torch.int32)[..., None] - 127)
        return torch.where((slots >= 0)[:, None, None], x, 0.0).to(DTYPES[c["dtype"]])

    return rows(st["k_cache"]), rows(st["v_cache"])


def _plain_attention(st):
    c = st["case"]
    q, lens, table = st["q"], st["kv_lens"].long(), st["page_table"].long()
    H, kv, dim, page = c["heads"], c["kv"], c["dim"], c["page"]
    B, mq, mk, dev = lens.numel(), st["max_q"], st["max_kv"], q.device
    T = q.shape[0]
    if st["cu_seqlens"] is None:
        seq, i = torch.arange(T, device=dev), torch.zeros(T, dtype=torch.long, device=dev)
        n = torch.ones(B, dtype=torch.long, device=dev)
    else:
        cu = st["cu_seqlens"].long()
        t = torch.arange(T, device=dev)
        seq = (t[:, None] >= cu[None, 1:]).sum(dim=1)
        i = t - cu[seq]
        n = cu[1:] - cu[:-1]
    padded = torch.zeros(B, mq, H, dim, device=dev)
    padded[seq, i] = q.float()
    pages = table[:, : -(-mk // page)]

    def gathered(cache):                                                 # [B, kv, keys, dim]
        return _dequantised(*cache, pages).permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :mk]

    # [B, kv, G * mq, dim] x [B, kv, dim, keys]
    G = H // kv
    rows = padded.unflatten(2, (kv, G)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    scores = torch.matmul(rows, gathered(st["k_cache"]).transpose(2, 3).contiguous()).unflatten(2, (G, mq))
    scores.mul_(st["scale"])
    j = torch.arange(mk, device=dev)
    p = (lens - n)[:, None] + torch.arange(mq, device=dev)[None, :]
    seen = (j[None, None, :] <= p[:, :, None]) & (j[None, None, :] < lens[:, None, None])
    if c["window"]:
        seen &= j[None, None, :] > p[:, :, None] - c["window"]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    scores.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    total = scores.sum(dim=-1, keepdim=True)
    out = torch.matmul(scores.flatten(2, 3), gathered(st["v_cache"]).contiguous()).unflatten(2, (G, mq))
    out = torch.where(total > 0, out / total, 0.0)                        # [B, kv, G, mq, dim]
    return out.permute(0, 3, 1, 2, 4).flatten(2, 3)[seq, i].to(q.dtype)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    kv, dim = case["kv"], case["dim"]
    row = dim + 1                                            # bytes of a quantised row
    if case["op"] == "append":
        T, R, H = case["tokens"], case["rot"], case["heads"]
        stored = 2 * kv * (row if case["quant"] else dim * e)
        return {"bytes": T * ((2 * H + 2 * kv) * dim * e + stored + 4 * R + 16) + (2 * dim * e if case["norm"] else 0),
                "flops": T * (3 * (H + kv) * R + (4 * (H + kv) * dim if case["norm"] else 0) + (2 * 2 * kv * dim if case["quant"] else 0))}
    if case["op"] == "read":
        return {"bytes": case["tokens"] * (2 * kv * (row + dim * e) + 8), "flops": case["tokens"] * 2 * kv * dim}
    H = case["heads"]
    n, length = _lengths(case)
    W = case["window"]
    keys = pairs = 0
    for m, L in zip(n, length):
        p = np.arange(L - m, L)
        first = np.maximum(0, p - W + 1) if W else np.zeros_like(p)
        seen = np.maximum(0, p + 1 - first)
        pairs += int(seen.sum())
        keys += L - int(first[0]) if L else 0
    return {"bytes": keys * kv * 2 * row + 2 * sum(n) * H * dim * e + 4 * sum(-(-x // case["page"]) for x in length),
            "flops": 4 * dim * H * pairs}


# ---------------------------------------------------------------------------
# From the definitions, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    page = case["page"]
    if case["op"] == "append":
        R = case["rot"]
        # each pair of columns as one complex number, turned by its position's angle
        turn = torch.complex(*st["cos_sin"].double()[st["positions"]].chunk(2, dim=1))[:, None, :]

        def rotated(x, w):
            x = x.double()
            x = x.clone() if w is None else x / (x.pow(2).sum(2) / x.shape[2] + EPS).sqrt()[..., None] * w.double()
            first, second = (slice(0, R // 2), slice(R // 2, R)) if case["style"] == "half" else (slice(0, R, 2), slice(1, R, 2))
            z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
            x[..., first], x[..., second] = z.real, z.imag
            return x

        live = torch.nonzero(st["slots"] >= 0).flatten()
        slot = st["slots"][live]

        def stored(cache, rows):
            rows = rows[live]
            if not case["quant"]:
                cache = cache.double()
                cache[slot // page, :, slot % page] = rows
                return cache
            values, scales = cache[0].double(), torch.exp2(cache[1].view(torch.uint8).double() - 127)
            e = torch.ceil(torch.log2(rows.abs().amax(2).clamp(min=2.0 ** -200) / 448)).clamp(min=-126)
            y = rows / torch.exp2(e)[..., None]
            # e4m3: three bits after the first one, steps of 2^-9 below 2^-6
            step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
            values[slot // page, :, slot % page] = torch.round(y / step) * step
            scales[slot // page, :, slot % page] = torch.exp2(e)
            return values, scales

        return (rotated(st["q"], st["q_norm"]), stored(st["k_cache"], rotated(st["k"], st["k_norm"])),
                stored(st["v_cache"], st["v"].double()))

    def row(cache, at, r):
        values, scales = (t.view(torch.uint8)[at, :, r] for t in cache)
        return values.view(E4M3).double() * torch.exp2(scales.double() - 127)[..., None]

    if case["op"] == "read":
        at = st["slots"].clamp(min=0)
        return tuple(row(st[c], at // page, at % page) * (st["slots"] >= 0)[:, None, None] for c in ("k_cache", "v_cache"))
    if work(case)["flops"] > 2.0e11:
        return None
    n, length = _lengths(case)
    H, kv, dim, W = case["heads"], case["kv"], case["dim"], case["window"]
    out = torch.zeros(sum(n), H, dim, dtype=torch.float64, device=st["q"].device)
    t = 0
    for s, (m, L) in enumerate(zip(n, length)):
        if L:
            j = torch.arange(L, device=out.device)
            k, v = (row(st[c], st["page_table"][s].long()[j // page], j % page) for c in ("k_cache", "v_cache"))  # [L, kv, dim]
            for at in range(0, m, 256):                          # rows of queries, to bound the scores
                q = st["q"][t + at: t + min(m, at + 256)].double().unflatten(1, (kv, H // kv))
                p = L - m + at + torch.arange(q.shape[0], device=out.device)
                hidden = j[None, :] > p[:, None]
                if W:
                    hidden |= j[None, :] <= p[:, None] - W
                for h in range(kv):
                    a = torch.tensordot(q[:, h], k[:, h], dims=([2], [1])) * dim ** -0.5
                    a = torch.softmax(a.masked_fill(hidden[:, None, :], -math.inf), dim=2)
                    out[t + at: t + at + q.shape[0], h * (H // kv): (h + 1) * (H // kv)] = torch.tensordot(a, v[:, h], dims=([2], [0]))
        t += m
    return out
