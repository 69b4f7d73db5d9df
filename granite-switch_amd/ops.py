"""``torch.ops.granite_switch.*`` registrations backed by the HIP library.

The reference registers its Triton launchers as custom ops in a dedicated
``granite_switch`` namespace so torch.compile / graph capture treat them as
opaque (src/granite_switch/vllm/core/lora_ops.py:25-27,192-226;
src/granite_switch/vllm/core/lora_kernel_meta.py:166-182).  This module
registers the same op names with the same argument lists, ``mutates_args`` and
fake implementations, so callers such as ``SwitchedLoRALinear._run_expand``
(src/granite_switch/vllm/core/lora.py:659-686) and ``WCrossShunt.forward``
(src/granite_switch/vllm/decoder/shadow_residual/wcross_shunt.py:198-242) run
unchanged on MI355X, plus three new ops for the y-given switched-LoRA path and
seven for the paged cache and the norms around the residual add.

Only one provider of the ``granite_switch`` ops can be loaded in a process.
"""

from __future__ import annotations

import torch

from . import kernels, norms, paged, switched

_NS = "granite_switch"


def _registered(name: str) -> bool:
    try:
        getattr(getattr(torch.ops, _NS), name)
        return True
    except (AttributeError, RuntimeError):
        return False


# ---------------------------------------------------------------------------
# Reference ops (same schemas)
# ---------------------------------------------------------------------------
if not _registered("switch_lora_expand"):

    @torch.library.custom_op(f"{_NS}::switch_lora_expand", mutates_args=("x_ext",))
    def switch_lora_expand(x_ext: torch.Tensor, adapter_indices: torch.Tensor, bitmask: torch.Tensor,
                           lb_packed: torch.Tensor, tile_slice: torch.Tensor, slice_col_r: torch.Tensor, NA_16: int,
                           NA_32: int, NA_64: int, NA_128: int, NA_256: int, NA_512: int, S: int, block_n: int,
                           N: int) -> None:
        kernels.switch_lora_expand(x_ext, adapter_indices, bitmask, lb_packed, tile_slice, slice_col_r,
                                   (NA_16, NA_32, NA_64, NA_128, NA_256, NA_512), S, block_n, N)

    @switch_lora_expand.register_fake
    def _(x_ext, adapter_indices, bitmask, lb_packed, tile_slice, slice_col_r, NA_16, NA_32, NA_64, NA_128, NA_256,
          NA_512, S, block_n, N):
        return None


if not _registered("switch_lora_expand_swiglu"):

    @torch.library.custom_op(f"{_NS}::switch_lora_expand_swiglu", mutates_args=("out",))
    def switch_lora_expand_swiglu(out: torch.Tensor, x_ext: torch.Tensor, adapter_indices: torch.Tensor,
                                  bitmask: torch.Tensor, lb_packed: torch.Tensor, slice_col_r: torch.Tensor,
                                  NA_16: int, NA_32: int, NA_64: int, NA_128: int, NA_256: int, NA_512: int, S: int,
                                  block_n: int, H: int, N: int) -> None:
        kernels.switch_lora_expand_swiglu(out, x_ext, adapter_indices, bitmask, lb_packed, slice_col_r,
                                          (NA_16, NA_32, NA_64, NA_128, NA_256, NA_512), S, block_n, H, N)

    @switch_lora_expand_swiglu.register_fake
    def _(out, x_ext, adapter_indices, bitmask, lb_packed, slice_col_r, NA_16, NA_32, NA_64, NA_128, NA_256, NA_512,
          S, block_n, H, N):
        return None


if not _registered("switch_lora_shrink_expand"):

    @torch.library.custom_op(f"{_NS}::switch_lora_shrink_expand", mutates_args=("out",))
    def switch_lora_shrink_expand(out: torch.Tensor, x_ext: torch.Tensor, adapter_indices: torch.Tensor,
                                  bitmask: torch.Tensor, lb_packed: torch.Tensor, tile_slice: torch.Tensor,
                                  slice_col_r: torch.Tensor, NA_16: int, NA_32: int, NA_64: int, NA_128: int,
                                  NA_256: int, NA_512: int, S: int, block_n: int, N: int) -> None:
        kernels.switch_lora_shrink_expand(out, x_ext, adapter_indices, bitmask, lb_packed, tile_slice, slice_col_r,
                                          (NA_16, NA_32, NA_64, NA_128, NA_256, NA_512), S, block_n, N)

    @switch_lora_shrink_expand.register_fake
    def _(out, x_ext, adapter_indices, bitmask, lb_packed, tile_slice, slice_col_r, NA_16, NA_32, NA_64, NA_128,
          NA_256, NA_512, S, block_n, N):
        return None


if not _registered("compute_per_module_bitmasks"):

    @torch.library.custom_op(f"{_NS}::compute_per_module_bitmasks", mutates_args=())
    def compute_per_module_bitmasks(adapter_indices: torch.Tensor, remap_tables_t: torch.Tensor) -> torch.Tensor:
        return kernels.compute_per_module_bitmasks(adapter_indices, remap_tables_t)

    @compute_per_module_bitmasks.register_fake
    def _(adapter_indices, remap_tables_t):
        M = adapter_indices.shape[0]
        num_modules = remap_tables_t.shape[1]
        bm = kernels.BLOCK_M
        return torch.empty(num_modules, (M + bm - 1) // bm, dtype=torch.int64, device=adapter_indices.device)


# ---------------------------------------------------------------------------
# y-given switched-LoRA ops
# ---------------------------------------------------------------------------
if not _registered("build_segments"):

    @torch.library.custom_op(f"{_NS}::build_segments", mutates_args=())
    def build_segments(adapter_ids: torch.Tensor, num_adapters: int, positions: torch.Tensor | None,
                       cu_seqlens: torch.Tensor | None,
                       act_offsets: torch.Tensor | None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        s = switched.build_segments(adapter_ids, num_adapters, positions, cu_seqlens, act_offsets)
        return s.eff_ids, s.seg_offsets, s.perm

    @build_segments.register_fake
    def _(adapter_ids, num_adapters, positions, cu_seqlens, act_offsets):
        T = adapter_ids.numel()
        dev = adapter_ids.device
        return (torch.empty(T, dtype=torch.int32, device=dev), torch.empty(num_adapters + 1, dtype=torch.int32, device=dev),
                torch.empty(max(T, 1), dtype=torch.int32, device=dev))


def _packed_view(a_pack, b_pack, a_off, b_off, ranks, slice_bounds, hidden, max_rank):
    out_slices = tuple(int(slice_bounds[i + 1] - slice_bounds[i]) for i in range(len(slice_bounds) - 1))
    return switched.PackedAdapters(a_pack=a_pack, b_pack=b_pack, a_off=a_off, b_off=b_off, ranks=ranks,
                                   ranks_host=[], output_slices=out_slices, hidden=int(hidden),
                                   num_adapters=int(ranks.numel() - 1), max_rank=int(max_rank))


def _segs(seg_offsets, perm, T):
    return switched.Segments(eff_ids=perm, seg_offsets=seg_offsets, perm=perm, num_tokens=int(T),
                             num_adapters=int(seg_offsets.numel() - 1))


if not _registered("switched_lora_shrink"):

    @torch.library.custom_op(f"{_NS}::switched_lora_shrink", mutates_args=())
    def switched_lora_shrink(x: torch.Tensor, seg_offsets: torch.Tensor, perm: torch.Tensor, a_pack: torch.Tensor,
                             a_off: torch.Tensor, ranks: torch.Tensor, num_slices: int, max_rank: int) -> torch.Tensor:
        bounds = list(range(num_slices + 1))   # only the slice count matters for the shrink
        pk = _packed_view(a_pack, a_pack, a_off, a_off, ranks, bounds, x.shape[-1], max_rank)
        return switched.shrink(x, _segs(seg_offsets, perm, x.shape[0]), pk)

    @switched_lora_shrink.register_fake
    def _(x, seg_offsets, perm, a_pack, a_off, ranks, num_slices, max_rank):
        return torch.empty(max(x.shape[0], 1), num_slices * max_rank, dtype=x.dtype, device=x.device)


if not _registered("switched_lora_expand_add"):

    @torch.library.custom_op(f"{_NS}::switched_lora_expand_add", mutates_args=("y",))
    def switched_lora_expand_add(y: torch.Tensor, z: torch.Tensor, seg_offsets: torch.Tensor, perm: torch.Tensor,
                                 b_pack: torch.Tensor, b_off: torch.Tensor, ranks: torch.Tensor,
                                 slice_bounds: list[int], max_rank: int) -> None:
        pk = _packed_view(b_pack, b_pack, b_off, b_off, ranks, slice_bounds, 0, max_rank)
        switched.expand_add_(y, z, _segs(seg_offsets, perm, y.shape[0]), pk)

    @switched_lora_expand_add.register_fake
    def _(y, z, seg_offsets, perm, b_pack, b_off, ranks, slice_bounds, max_rank):
        return None


# ---------------------------------------------------------------------------
# The paged cache and the residual stream
# ---------------------------------------------------------------------------
if not _registered("cache_slots"):

    @torch.library.custom_op(f"{_NS}::cache_slots", mutates_args=())
    def cache_slots(page_table: torch.Tensor, kv_lens: torch.Tensor, page_size: int, num_pages: int,
                    cu_seqlens: torch.Tensor | None, num_tokens: int) -> tuple[torch.Tensor, torch.Tensor]:
        return paged.cache_slots(page_table, kv_lens, page_size, num_pages, cu_seqlens, num_tokens)

    @cache_slots.register_fake
    def _(page_table, kv_lens, page_size, num_pages, cu_seqlens, num_tokens):
        return (torch.empty(num_tokens, dtype=torch.int64, device=kv_lens.device),
                torch.empty(num_tokens, dtype=torch.int64, device=kv_lens.device))


if not _registered("append_kv"):

    @torch.library.custom_op(f"{_NS}::append_kv", mutates_args=("k_cache", "v_cache"))
    def append_kv(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  slots: torch.Tensor, positions: torch.Tensor | None, cos_sin: torch.Tensor | None,
                  interleaved: bool) -> torch.Tensor:
        with torch.no_grad():          # autograd is the op's: a backward through it raises
            return paged.append_kv_(q, k, v, k_cache, v_cache, slots, positions, cos_sin, interleaved=interleaved)

    @append_kv.register_fake
    def _(q, k, v, k_cache, v_cache, slots, positions, cos_sin, interleaved):
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)


def _cache(values: torch.Tensor, scales: torch.Tensor | None):
    return values if scales is None else paged.QuantizedCache(values, scales)


if not _registered("append_kv_normed"):

    @torch.library.custom_op(f"{_NS}::append_kv_normed", mutates_args=("k_cache", "v_cache", "k_scales", "v_scales"))
    def append_kv_normed(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                         k_scales: torch.Tensor | None, v_scales: torch.Tensor | None, slots: torch.Tensor,
                         positions: torch.Tensor | None, cos_sin: torch.Tensor | None, interleaved: bool,
                         q_norm: torch.Tensor | None, k_norm: torch.Tensor | None, eps: float) -> torch.Tensor:
        with torch.no_grad():          # autograd is the op's: a backward through it raises
            return paged.append_kv_(q, k, v, _cache(k_cache, k_scales), _cache(v_cache, v_scales), slots, positions, cos_sin,
                                    interleaved=interleaved, q_norm=q_norm, k_norm=k_norm, eps=eps)

    @append_kv_normed.register_fake
    def _(q, k, v, k_cache, v_cache, k_scales, v_scales, slots, positions, cos_sin, interleaved, q_norm, k_norm, eps):
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)


if not _registered("read_kv"):

    @torch.library.custom_op(f"{_NS}::read_kv", mutates_args=())
    def read_kv(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scales: torch.Tensor | None, v_scales: torch.Tensor | None,
                slots: torch.Tensor, dtype: torch.dtype | None) -> tuple[torch.Tensor, torch.Tensor]:
        with torch.no_grad():          # autograd is the op's: a backward through it raises
            return paged.read_kv(_cache(k_cache, k_scales), _cache(v_cache, v_scales), slots, dtype)

    @read_kv.register_fake
    def _(k_cache, v_cache, k_scales, v_scales, slots, dtype):
        dtype = dtype or (k_cache.dtype if k_scales is None else torch.bfloat16)
        shape = (slots.shape[0], k_cache.shape[1], k_cache.shape[3])
        return torch.empty(shape, dtype=dtype, device=slots.device), torch.empty(shape, dtype=dtype, device=slots.device)


if not _registered("paged_attention_e4m3"):

    @torch.library.custom_op(f"{_NS}::paged_attention_e4m3", mutates_args=())
    def paged_attention_e4m3(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scales: torch.Tensor,
                             v_scales: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor,
                             cu_seqlens: torch.Tensor | None, scale: float | None, window: int,
                             max_q: int | None) -> torch.Tensor:
        with torch.no_grad():          # autograd is the op's: a backward through it raises
            return paged.paged_attention(q, _cache(k_cache, k_scales), _cache(v_cache, v_scales), page_table, kv_lens,
                                         cu_seqlens, scale, window, max_q=max_q)

    @paged_attention_e4m3.register_fake
    def _(q, k_cache, v_cache, k_scales, v_scales, page_table, kv_lens, cu_seqlens, scale, window, max_q):
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)


if not _registered("paged_attention"):

    @torch.library.custom_op(f"{_NS}::paged_attention", mutates_args=())
    def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                        kv_lens: torch.Tensor, cu_seqlens: torch.Tensor | None, scale: float | None, window: int,
                        max_q: int | None) -> torch.Tensor:
        with torch.no_grad():          # autograd is the op's: a backward through it raises
            return paged.paged_attention(q, k_cache, v_cache, page_table, kv_lens, cu_seqlens, scale, window, max_q=max_q)

    @paged_attention.register_fake
    def _(q, k_cache, v_cache, page_table, kv_lens, cu_seqlens, scale, window, max_q):
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)


if not _registered("residual_norm"):

    @torch.library.custom_op(f"{_NS}::residual_norm", mutates_args=())
    def residual_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float, scale: float,
                      gate: torch.Tensor | None, post_weight: torch.Tensor | None,
                      gate_act: str | None) -> tuple[torch.Tensor, torch.Tensor]:
        with torch.no_grad():          # autograd is the op's: a backward through it raises
            return norms.residual_norm(x, residual, weight, eps, scale, gate, post_weight, gate_act)

    @residual_norm.register_fake
    def _(x, residual, weight, eps, scale, gate, post_weight, gate_act):
        return (torch.empty(x.shape, dtype=x.dtype, device=x.device),
                torch.empty(residual.shape, dtype=residual.dtype, device=residual.device))


def op(name: str):
    """``torch.ops.granite_switch.<name>``."""
    return getattr(getattr(torch.ops, _NS), name)
