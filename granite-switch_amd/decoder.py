"""A switched-LoRA decoder over a paged cache: the operators of this package, put together.

One layer, for the rows of a step (decode rows, chunks of prompts, the few
invocation tokens of an adapter that switches on mid-sequence, in one batch):

    y, r = residual_norm(x, r, input_norm, scale=m)      the block before, the residual stream, the norm
    q, k, v = qkv(y)                                     switched projection, slices of its output
    q = append_kv_(q, k, v, cache, slots, positions)     normed, rotated; keys and values stored
    o = paged_attention(q, cache, page_table, kv_lens)   this step's tokens included
    y, r = residual_norm(o_proj(o), r, mlp_norm, scale=m)
    x = down(swiglu(gate_up(y)))                         switched projections

The arrangement is Granite's: ``residual_multiplier`` scales each block's output
and ``attention_multiplier`` the scores.  ``PagedStep`` holds what all layers of a
step share; ``LoRAContext`` the step's routing.

    decoder = SwitchedDecoder(layers, final_norm, num_adapters); decoder.finalize(adapter_ranks)
    step = PagedStep(page_table, kv_lens, page_size, num_pages, rope, cu_seqlens, num_tokens)
    decoder.route(adapter_ids, step.positions, cu_seqlens, act_offsets)
    hidden = decoder(embeddings, step, caches)
"""

from __future__ import annotations

import torch
from torch import nn

from . import norms, paged
from .meta import FusedLoRAKernelMeta, LoRAContext
from .vllm_layers import SwitchedLoRALinear


class PagedStep:
    """One step's batch: its pages, lengths, rows, slots and positions; computed once for all layers."""

    __slots__ = ("cos_sin", "cu_seqlens", "kv_lens", "max_q", "page_table", "positions", "slots")

    def __init__(self, page_table: torch.Tensor, kv_lens: torch.Tensor, page_size: int, num_pages: int,
                 cos_sin: torch.Tensor | None, cu_seqlens: torch.Tensor | None = None, num_tokens: int | None = None,
                 max_q: int | None = None):
        self.page_table, self.kv_lens, self.cu_seqlens = page_table, kv_lens, cu_seqlens
        self.cos_sin, self.max_q = cos_sin, max_q
        self.slots, self.positions = paged.cache_slots(page_table, kv_lens, page_size, num_pages, cu_seqlens, num_tokens)


class SwitchedDecoderLayer(nn.Module):
    """Attention and MLP blocks whose four projections are ``SwitchedLoRALinear``.

    ``qkv`` has three slices (heads * head_dim, kv_heads * head_dim twice),
    ``gate_up`` two with ``fuse_swiglu``; ``window`` > 0 is a sliding window.
    ``q_norm`` and ``k_norm`` [head_dim] norm each head before its rotation.  The
    cache is a pair of tensors or of ``paged.QuantizedCache``, of a head_dim and page
    size that ``paged.paged_attention`` takes.
    """

    def __init__(self, qkv: SwitchedLoRALinear, o_proj: SwitchedLoRALinear, gate_up: SwitchedLoRALinear,
                 down: SwitchedLoRALinear, input_norm: torch.Tensor, mlp_norm: torch.Tensor, heads: int, kv_heads: int,
                 head_dim: int, eps: float = 1e-5, residual_multiplier: float = 1.0,
                 attention_multiplier: float | None = None, window: int = 0, q_norm: torch.Tensor | None = None,
                 k_norm: torch.Tensor | None = None):
        super().__init__()
        widths = (heads * head_dim, kv_heads * head_dim, kv_heads * head_dim)
        if qkv.output_slices != widths:
            raise ValueError(f"SwitchedDecoderLayer: qkv has slices {qkv.output_slices}, {heads} query and {kv_heads} "
                             f"key/value heads of {head_dim} need {widths}")
        if not gate_up.fuse_swiglu:
            raise ValueError("SwitchedDecoderLayer: gate_up needs fuse_swiglu")
        self.qkv, self.o_proj, self.gate_up, self.down = qkv, o_proj, gate_up, down
        self.register_buffer("input_norm", input_norm.detach())
        self.register_buffer("mlp_norm", mlp_norm.detach())
        for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
            if w is not None and tuple(w.shape) != (head_dim,):
                raise ValueError(f"SwitchedDecoderLayer: {name} is {tuple(w.shape)}, heads of {head_dim}")
            self.register_buffer(name, None if w is None else w.detach())
        self.heads, self.kv_heads, self.head_dim, self.eps = heads, kv_heads, head_dim, eps
        self.residual_multiplier, self.attention_multiplier, self.window = residual_multiplier, attention_multiplier, window

    def linears(self) -> list:
        return [self.qkv, self.o_proj, self.gate_up, self.down]

    def forward(self, x: torch.Tensor | None, residual: torch.Tensor, step: PagedStep,
                cache: tuple) -> tuple[torch.Tensor, torch.Tensor]:
        """``(x, residual)`` [T, hidden]: the block before and the stream (x None: the first layer), and after."""
        paged.check_attended(*cache)                       # before a row is stored
        T, D = residual.shape[0], self.head_dim
        y, residual = norms.residual_norm(x, residual, self.input_norm, self.eps, self.residual_multiplier)
        qkv = self.qkv(y)[0]
        nq, nk = self.heads * D, self.kv_heads * D
        q, k, v = (qkv[:, a:b].unflatten(1, (-1, D)) for a, b in ((0, nq), (nq, nq + nk), (nq + nk, nq + 2 * nk)))
        q = paged.append_kv_(q, k, v, *cache, step.slots, step.positions, step.cos_sin, q_norm=self.q_norm,
                             k_norm=self.k_norm, eps=self.eps)
        o = paged.paged_attention(q, *cache, step.page_table, step.kv_lens, step.cu_seqlens, self.attention_multiplier,
                                  self.window, max_q=step.max_q)
        y, residual = norms.residual_norm(self.o_proj(o.view(T, nq))[0], residual, self.mlp_norm, self.eps,
                                          self.residual_multiplier)
        return self.down(self.gate_up(y)[0])[0], residual


class SwitchedDecoder(nn.Module):
    """Layers that share one routing, then the last residual add and norm."""

    def __init__(self, layers: list, final_norm: torch.Tensor, num_adapters: int):
        super().__init__()
        self.layers = nn.ModuleList(layers)
        self.register_buffer("final_norm", final_norm.detach())
        self.num_adapters = num_adapters
        self.ctx = LoRAContext()
        self.meta = FusedLoRAKernelMeta(final_norm.device)

    def finalize(self, adapter_ranks: list) -> None:
        """Lay the weights out and number the projections; once, after loading."""
        tables, keys = [], []
        for layer in self.layers:
            for lin in layer.linears():
                lin.finalize_weights(adapter_ranks)
                lin._module_idx = len(tables)
                lin._lora_ctx = self.ctx
                tables.append(lin.remap_table)
                keys.append(lin._block_cfg_key)
        self.meta.register_remap_tables(torch.stack(tables), keys)

    def route(self, adapter_ids: torch.Tensor, positions: torch.Tensor | None = None,
              cu_seqlens: torch.Tensor | None = None, act_offsets: torch.Tensor | None = None) -> None:
        """Each row's adapter (0: the base model) for the steps that follow; ``act_offsets`` as ``build_segments`` has them."""
        self.meta.prepare_and_store(adapter_ids, self.ctx, positions, cu_seqlens, act_offsets)

    def forward(self, embeddings: torch.Tensor, step: PagedStep, caches: list) -> torch.Tensor:
        """Normed hidden states [T, hidden] of the step's rows; ``caches``: a (key, value) pair per layer."""
        x, residual = None, embeddings
        for layer, cache in zip(self.layers, caches, strict=True):
            x, residual = layer(x, residual, step, cache)
        last = self.layers[-1]
        return norms.residual_norm(x, residual, self.final_norm, last.eps, last.residual_multiplier)[0]


__all__ = ["PagedStep", "SwitchedDecoder", "SwitchedDecoderLayer"]
