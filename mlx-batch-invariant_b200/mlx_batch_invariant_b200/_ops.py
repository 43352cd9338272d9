"""torch.library registrations of the invariant operators, so torch.compile sees each
as one opaque op (the reference's kernels are likewise opaque to mx.compile).

Eager calls go straight to libbi.so; under torch.compile the public functions call
these ops, whose real implementation is that same eager path -- the bits are the
same either way.  The fake implementations give the output's shape and dtype only.
"""

from typing import List, Optional, Tuple

import torch

_NS = "mlx_bi"


@torch.library.custom_op(_NS + "::gemm", mutates_args=())
def gemm(a: torch.Tensor, b: torch.Tensor, bias: Optional[torch.Tensor], transpose_b: bool,
         alpha: float, beta: float) -> torch.Tensor:
    """bi_gemm: alpha * (a @ B) + beta * bias with B = b.T if transpose_b else b."""
    from ._gemm import _gemm_eager
    return _gemm_eager(a, b, bias, transpose_b, alpha, beta)


@gemm.register_fake
def _gemm_fake(a, b, bias, transpose_b, alpha, beta):
    n = b.shape[0] if transpose_b else b.shape[1]
    return a.new_empty((*a.shape[:-1], n))


@torch.library.custom_op(_NS + "::sdpa", mutates_args=())
def sdpa(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, mask_mode: int,
         causal_offset: int, mask: Optional[torch.Tensor], mask_strides: List[int],
         sinks: Optional[torch.Tensor]) -> torch.Tensor:
    """bi_sdpa on validated arguments (see _attention._sdpa)."""
    from ._attention import _sdpa_eager
    return _sdpa_eager(q, k, v, scale, mask_mode, causal_offset, mask, mask_strides, sinks)


@sdpa.register_fake
def _sdpa_fake(q, k, v, scale, mask_mode, causal_offset, mask, mask_strides, sinks):
    return q.new_empty((q.shape[0], q.shape[1], q.shape[2], v.shape[3]))


@torch.library.custom_op(_NS + "::paged_plan", mutates_args=("block_table",))
def paged_plan(query_lens: torch.Tensor, context_lens: torch.Tensor, block_table: torch.Tensor,
               page_size: int, num_tokens: int, free_pages: Optional[torch.Tensor],
               free_head: Optional[torch.Tensor]) -> Tuple[
                   torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """bi_paged_plan on validated arguments (see _paged.paged_plan); an op returns tensors
    only, so without free pages the fifth is empty."""
    from ._paged import _plan_eager
    out = _plan_eager(query_lens, context_lens, block_table, page_size, num_tokens, free_pages,
                      free_head, query_lens.device)
    return (*out[:4], out[4] if out[4] is not None else query_lens.new_empty((0,)))


@paged_plan.register_fake
def _paged_plan_fake(query_lens, context_lens, block_table, page_size, num_tokens, free_pages,
                     free_head):
    R = query_lens.shape[0]
    long = torch.int64
    return (query_lens.new_empty((R + 1,)), query_lens.new_empty((R,)),
            query_lens.new_empty((num_tokens,), dtype=long),
            query_lens.new_empty((num_tokens,), dtype=long),
            query_lens.new_empty((1 if free_pages is not None else 0,)))


@torch.library.custom_op(_NS + "::rope_kv_paged", mutates_args=("k_cache", "v_cache"))
def rope_kv_paged(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                  positions: torch.Tensor, slots: torch.Tensor, k_cache: torch.Tensor,
                  v_cache: torch.Tensor) -> torch.Tensor:
    """bi_rope_kv_paged on validated arguments (see _paged.rope_kv_paged)."""
    from ._paged import _rope_eager
    return _rope_eager(qkv, cos, sin, positions, slots, k_cache, v_cache, None, qkv.device)


@rope_kv_paged.register_fake
def _rope_kv_paged_fake(qkv, cos, sin, positions, slots, k_cache, v_cache):
    hk, hd = k_cache.shape[1], k_cache.shape[3]
    return qkv.new_empty((qkv.shape[0], qkv.shape[1] // hd - 2 * hk, hd))


@torch.library.custom_op(_NS + "::paged_attention", mutates_args=())
def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    block_table: torch.Tensor, query_start: torch.Tensor,
                    seq_lens: torch.Tensor, scale: float, window: int, first_tokens: int,
                    sinks: Optional[torch.Tensor]) -> torch.Tensor:
    """bi_paged_sdpa on validated arguments (see _paged.paged_attention)."""
    from . import _lib
    from ._paged import _attention_eager
    return _attention_eager(q, k_cache, v_cache, block_table, query_start, seq_lens, scale,
                            window, first_tokens, sinks, None, _lib.dtype_code(q.dtype), q.device)


@paged_attention.register_fake
def _paged_attention_fake(q, k_cache, v_cache, block_table, query_start, seq_lens, scale,
                          window, first_tokens, sinks):
    return q.new_empty(q.shape)
