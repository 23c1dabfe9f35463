"""Operator surface with the reference's names and signatures
(reference: deepseek_v4_kernel/ops.py:17-72).  These are thin pass-throughs to
`deepseek_v4_kernel.cuda`; importing this module fails if the native library
has not been built."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

try:
    from . import cuda as _cuda
except ImportError as exc:  # pragma: no cover
    raise ImportError(
        "deepseek_v4_kernel native library not built: run build_native.py in the package "
        "directory (or __graft_entry__.build() at the repository root).") from exc


def sparse_decode_fwd(
    q: torch.Tensor,
    kv: torch.Tensor,
    indices: torch.Tensor,
    topk_length: Optional[torch.Tensor],
    attn_sink: Optional[torch.Tensor],
    tile_scheduler_metadata: Optional[torch.Tensor],
    num_splits: Optional[torch.Tensor],
    extra_kv: Optional[torch.Tensor],
    extra_indices: Optional[torch.Tensor],
    extra_topk_length: Optional[torch.Tensor],
    d_v: int,
    sm_scale: float,
) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """FlashMLA-compatible sparse decode: returns (out, lse[b, h_q, s_q],
    tile_scheduler_metadata, num_splits)."""
    return _cuda.sparse_decode_fwd(q, kv, indices, topk_length, attn_sink,
                                   tile_scheduler_metadata, num_splits, extra_kv, extra_indices,
                                   extra_topk_length, int(d_v), float(sm_scale))


def sparse_prefill_fwd(
    q: torch.Tensor,
    kv: torch.Tensor,
    indices: torch.Tensor,
    sm_scale: float,
    d_v: int = 512,
    attn_sink: Optional[torch.Tensor] = None,
    topk_length: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Drop-in for ``sgl_kernel.flash_mla.flash_mla_sparse_fwd``: flat BF16 kv,
    returns (out, max_logits, lse)."""
    return _cuda.sparse_prefill_fwd(q, kv, indices, float(sm_scale), int(d_v), attn_sink,
                                    topk_length)


def sparse_prefill_fwd_fp8(q, kv, indices, sm_scale, d_v=512, attn_sink=None, topk_length=None):
    """Prefill straight from the FP8 paged cache (same returns as sparse_prefill_fwd)."""
    return _cuda.sparse_prefill_fwd_fp8(q, kv, indices, float(sm_scale), int(d_v), attn_sink,
                                        topk_length)


def shared_prefix_decode_fwd(q, kv, prefix_table, prefix_length, block_table, suffix_length, attn_sink, d_v, sm_scale):
    """Dense decode of a batch that shares a long prefix over the FP8 paged cache, the prefix
    attended once for all requests: returns (out, lse[b, h_q, s_q])."""
    return _cuda.shared_prefix_decode_fwd(q, kv, prefix_table, prefix_length, block_table, suffix_length, attn_sink,
                                          int(d_v), float(sm_scale))


def dense_prefill_fwd(q, k, v, cu_seqlens_q, cu_seqlens_k, sm_scale, causal=True, attn_sink=None, out=None):
    """Dense causal attention of packed sequences with grouped heads (prompts, chunks behind a
    context, single tokens): the same returns as sparse_prefill_fwd."""
    return _cuda.dense_prefill_fwd(q, k, v, cu_seqlens_q, cu_seqlens_k, float(sm_scale), causal, attn_sink, out)


def kv_store(k_nope, k_rope, slots, kv) -> None:
    """Quantise BF16 latent + RoPE rows into the FP8 paged cache at `slots`."""
    _cuda.kv_store(k_nope, k_rope, slots, kv)


def kv_store_rows(k, loc, kv) -> None:
    """The same store for the operands a serving framework's cache writer holds: one BF16
    row per token (latent then RoPE values, possibly a strided view) and its int32 / int64
    slot mapping."""
    _cuda.kv_store_rows(k, loc, kv)


def build_slot_maps(block_table, cached_lens, new_lens, free_pages, page_block, n_slots):
    """Extend block tables (in place) by the pages of this step's new tokens and map the
    tokens to cache slots, from request lengths on the device: returns (slots, positions,
    cu_new, cu_total, n_taken)."""
    return _cuda.build_slot_maps(block_table, cached_lens, new_lens, free_pages, page_block, n_slots)


def page_indices(block_table, positions, page_block, cu_seqlens=None) -> torch.Tensor:
    """Logical positions (an indexer's top-k lists) -> the physical token indices
    `sparse_decode_fwd` and the sparse prefills take."""
    return _cuda.page_indices(block_table, positions, page_block, cu_seqlens)
