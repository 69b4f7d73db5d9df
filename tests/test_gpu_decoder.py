"""GPU parity of the decoder put together over the paged cache, and of the registered ops.

The decoder's reference is a float64 restatement, token by token of each
sequence, from the bf16 weights.  Tolerance, on each row's relative error in the
2-norm: a layer rounds to bf16 (2^-8) 16 times on the way of a value (the two
norms' results and the two residuals; each projection's product and its sum with
the adapter; rotation; probabilities; attention; the gated product), two layers
and the last norm 33 times.  The roundings are independent and a block at most
doubles a relative error of its input (unit-scale weights; a product of two
factors): sqrt(33) 2^-8 2 = 4.5e-2.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from granite_switch_amd import decoder, norms, ops, paged, vllm_layers

pytestmark = pytest.mark.gpu

TOL = math.sqrt(33) * 2.0 ** -8 * 2
BF16 = torch.bfloat16
HIDDEN, HEADS, KV, DIM, MLP = 256, 8, 2, 64, 512
RANKS = [16, 32, 16]
EPS, RES, SCALE = 1e-5, 0.5, 1.0 / 64


def _say(msg):
    print(msg, flush=True)


def _linear(dev, g, n_in, slices, fuse=False):
    base = torch.nn.Linear(n_in, sum(slices), bias=False).to(device=dev, dtype=BF16)
    base.weight.data = (torch.randn(sum(slices), n_in, generator=g, device=dev) / n_in ** 0.5).to(BF16)
    lin = vllm_layers.SwitchedLoRALinear(base, len(RANKS), max(RANKS), num_slices=len(slices),
                                         output_slices=slices if len(slices) > 1 else None, fuse_swiglu=fuse)
    As = [lin.lora_A] if len(slices) == 1 else list(lin.lora_A_slices)
    Bs = [lin.lora_B] if len(slices) == 1 else list(lin.lora_B_slices)
    for s, width in enumerate(slices):
        for a, r in enumerate(RANKS):
            As[s].data[a, 0, :r] = (torch.randn(r, n_in, generator=g, device=dev) / n_in ** 0.5).to(BF16)
            Bs[s].data[a, 0, :, :r] = (0.1 * torch.randn(width, r, generator=g, device=dev)).to(BF16)
    f = lambda t: t.data.double().cpu().clone()
    return lin, (f(base.weight), [f(a) for a in As], [f(b) for b in Bs])


def _lin_ref(w, x, ids):
    W, As, Bs = w
    y = x @ W.T
    at = 0
    for A, B in zip(As, Bs):
        for i in np.unique(ids):
            if i:
                rows = torch.tensor(ids == i)
                y[rows, at:at + B.shape[2]] += x[rows] @ A[i - 1, 0].T @ B[i - 1, 0].T
        at += B.shape[2]
    return y


def _rms(x, w):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _rotate(x, pos, table):
    half = table.shape[1] // 2
    c, s = table[pos, None, :half], table[pos, None, half:]
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


class Reference:
    def __init__(self, layers, final, table, window):
        self.layers, self.final, self.table, self.window = layers, final, table, window
        self.kv = [dict() for _ in layers]

    def step(self, emb, n, ids):
        """emb [T, hidden], n rows of each sequence, ids [T]."""
        x, r = None, emb
        for L, kv in zip(self.layers, self.kv):
            r = r if x is None else r + RES * x
            qkv = _lin_ref(L["qkv"], _rms(r, L["input_norm"]), ids)
            T = r.shape[0]
            q, k, v = (t.reshape(T, -1, DIM) for t in qkv.split([HEADS * DIM, KV * DIM, KV * DIM], 1))
            o = torch.zeros(T, HEADS, DIM, dtype=torch.float64)
            at = 0
            for s, m in enumerate(n):
                if m == 0:
                    continue
                old = kv.get(s, (torch.zeros(0, KV, DIM).double(),) * 2)
                p = torch.arange(m) + old[0].shape[0]
                K = torch.cat([old[0], _rotate(k[at:at + m], p, self.table)])
                V = torch.cat([old[1], v[at:at + m]])
                kv[s] = (K, V)
                j = torch.arange(K.shape[0])
                seen = j[None] <= p[:, None]
                if self.window:
                    seen &= j[None] > p[:, None] - self.window
                Q = _rotate(q[at:at + m], p, self.table)
                for h in range(HEADS):
                    S = (Q[:, h] @ K[:, h // (HEADS // KV)].T * SCALE).masked_fill(~seen, -math.inf)
                    o[at:at + m, h] = torch.softmax(S, -1) @ V[:, h // (HEADS // KV)]
                at += m
            r = r + RES * _lin_ref(L["o_proj"], o.reshape(T, -1), ids)
            gu = _lin_ref(L["gate_up"], _rms(r, L["mlp_norm"]), ids)
            x = _lin_ref(L["down"], torch.nn.functional.silu(gu[:, :MLP]) * gu[:, MLP:], ids)
        return _rms(r + RES * x, self.final)


@pytest.mark.parametrize("window", [0, 50])
def test_decoder_steps(dev, window):
    g = torch.Generator(device=dev).manual_seed(3)
    widths = (HEADS * DIM, KV * DIM, KV * DIM)
    layers, refs = [], []
    norm = lambda: (1 + 0.2 * torch.randn(HIDDEN, generator=g, device=dev)).to(BF16)
    for _ in range(2):
        parts = {"qkv": _linear(dev, g, HIDDEN, widths), "o_proj": _linear(dev, g, HEADS * DIM, (HIDDEN,)),
                 "gate_up": _linear(dev, g, HIDDEN, (MLP, MLP), True), "down": _linear(dev, g, MLP, (HIDDEN,))}
        w = {"input_norm": norm(), "mlp_norm": norm()}
        layers.append(decoder.SwitchedDecoderLayer(**{k: v[0] for k, v in parts.items()}, **w, heads=HEADS, kv_heads=KV,
                                                   head_dim=DIM, eps=EPS, residual_multiplier=RES,
                                                   attention_multiplier=SCALE, window=window))
        refs.append({**{k: v[1] for k, v in parts.items()}, **{k: v.double().cpu() for k, v in w.items()}})
    final = norm()
    dec = decoder.SwitchedDecoder(layers, final, len(RANKS))
    dec.finalize(RANKS)
    table = paged.rope_table(512, DIM, device=dev)
    ref = Reference(refs, final.double().cpu(), table.double().cpu(), window)

    page, pages, B = 16, 64, 4
    pages_of = torch.randperm(pages, generator=g, device=dev)[: B * 12].view(B, 12).to(torch.int32)
    caches = [paged.allocate_cache(pages, KV, page, DIM, BF16, dev) for _ in layers]
    for pair in caches:
        for c in pair:
            c.fill_(math.nan)                             # rows that were never stored must not matter
    lens = np.zeros(B, np.int64)
    # prompts; decode rows beside a chunk of an adapter's tokens and a sequence without rows; decode rows
    steps = [([37, 5, 130, 1], False), ([1, 1, 20, 0], False), ([1, 1, 1, 1], True)]
    for n, decode in steps:
        T = sum(n)
        lens += n
        _say(f"decoder window={window} rows={n}")
        ids = torch.randint(0, len(RANKS) + 1, (T,), generator=g, device=dev)
        emb = torch.randn(T, HIDDEN, generator=g, device=dev).to(BF16)
        cu = None if decode else torch.tensor(np.concatenate([[0], np.cumsum(n)]), dtype=torch.int32, device=dev)
        step = decoder.PagedStep(pages_of, torch.tensor(lens, dtype=torch.int32, device=dev), page, pages, table, cu, T,
                                 None if decode else max(n))
        dec.route(ids)
        got = dec(emb, step, caches).double().cpu()
        want = ref.step(emb.double().cpu(), n, ids.cpu().numpy())
        err = ((got - want).norm(dim=1) / want.norm(dim=1)).max().item()
        assert err <= TOL, f"rows {n}: relative error {err:.3e}"
        base = ref.layers[0]["qkv"]
        if (ids > 0).any():                                # the adapters matter by more than the tolerance
            x = emb.double().cpu()
            moved = (_lin_ref(base, x, ids.cpu().numpy()) - x @ base[0].T)[(ids > 0).cpu()]
            assert moved.norm() > 2 * TOL * (x @ base[0].T).norm(dim=1).mean()


def test_registered_ops_match_the_functions(dev):
    g = torch.Generator(device=dev).manual_seed(9)
    B, page, pages, n = 3, 16, 24, [1, 9, 30]
    _say("registered ops of the paged cache and the norms")
    T = sum(n)
    lens = torch.tensor([50, 9, 100], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 1, 10, 40], dtype=torch.int32, device=dev)
    table = torch.randperm(pages, generator=g, device=dev).view(B, 8).to(torch.int32)
    slots, pos = ops.op("cache_slots")(table, lens, page, pages, cu, T)
    want_slots, want_pos = paged.cache_slots(table, lens, page, pages, cu, T)
    assert torch.equal(slots, want_slots) and torch.equal(pos, want_pos)
    qkv = torch.randn(T, HEADS + 2 * KV, DIM, generator=g, device=dev).to(BF16)
    q, k, v = qkv.split([HEADS, KV, KV], 1)
    rope = paged.rope_table(128, DIM, device=dev)
    c1 = [torch.randn(pages, KV, page, DIM, generator=g, device=dev).to(BF16) for _ in range(2)]
    c2 = [c.clone() for c in c1]
    q1 = ops.op("append_kv")(q, k, v, *c1, slots, pos, rope, False)
    q2 = paged.append_kv_(q, k, v, *c2, slots, pos, rope)
    assert torch.equal(q1, q2) and all(torch.equal(a, b) for a, b in zip(c1, c2))
    o1 = ops.op("paged_attention")(q1, *c1, table, lens, cu, None, 0, max(n))
    o2 = paged.paged_attention(q2, *c2, table, lens, cu, max_q=max(n))
    assert torch.equal(o1, o2)
    x, r = (torch.randn(T, HIDDEN, generator=g, device=dev).to(BF16) for _ in range(2))
    w = torch.randn(HIDDEN, generator=g, device=dev).to(BF16)
    gate = torch.randn(T, 1, generator=g, device=dev).to(BF16)
    for a, b in zip(ops.op("residual_norm")(x, r, w, EPS, RES, gate, w, "sigmoid"),
                    norms.residual_norm(x, r, w, EPS, RES, gate, w, "sigmoid")):
        assert torch.equal(a, b)
