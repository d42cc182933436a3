"""algebraic_intelligence_amd — Algebraic FlashAttention (AFA) for AMD MI355X (gfx950).

A drop-in for the AFA hot path of tasmaikeni13/algebraic-intelligence: the fused forward
(pallas_afa_forward / tiled_afa_forward), its analytical backward (pallas_afa custom VJP),
the padding front door (algebraic_flash_attention), the sequence ring (distributed_ring_afa, its
hops run in turn on one GPU) and the batch x heads placement (sharded_pallas_afa), the A-Softmax (algebraic_softmax), the
octic weight (octic_kernel), the Cayley rotary (AGO) tables and rotation, the OACE loss head
(fused_linear_oace, fused_oace_softmax_loss), and serving over a paged cache (PagePool, DraftPlan,
build_block_tables, append_to_cache, paged_tree_afa, and paged_prefix_afa behind a prefix that all requests share) with
positions of several axes (apply_ago_axis_rotations) and norms of q and k (apply_ago_norm_rotations), and a cache cut back
to the tokens that attention gives most (accumulate_cache_weights, evict_from_cache) — all running in hand-written HIP kernels behind the C ABI of include/afa.h.
"""
from .afa import (
    afa_flops,
    algebraic_flash_attention,
    distributed_ring_afa,
    exact_afa_reference,
    exact_afa_with_denominator,
    pallas_afa,
    pallas_afa_forward,
    sharded_pallas_afa,
    tiled_afa_backward,
    tiled_afa_forward,
)
from .attention import (
    CayleyRotary,
    algebraic_softmax,
    apply_ago_axis_rotations,
    apply_ago_norm_rotations,
    apply_ago_rotations,
    build_cayley_rotary_matrix,
    octic_kernel,
    rotate_tensor,
)
from .eviction import (
    accumulate_cache_weights,
    evict_from_cache,
)
from .paged import (
    DraftPlan,
    PagePool,
    append_to_cache,
    build_block_tables,
    paged_prefix_afa,
    paged_tree_afa,
)
from .oace import (
    fused_linear_oace,
    fused_linear_oace_backward,
    fused_linear_oace_forward,
    fused_oace_softmax_loss,
)

__all__ = [
    "afa_flops", "algebraic_flash_attention", "distributed_ring_afa", "exact_afa_reference", "exact_afa_with_denominator",
    "pallas_afa", "pallas_afa_forward", "sharded_pallas_afa", "tiled_afa_backward", "tiled_afa_forward",
    "CayleyRotary", "algebraic_softmax", "apply_ago_axis_rotations", "apply_ago_rotations", "build_cayley_rotary_matrix",
    "octic_kernel", "rotate_tensor", "fused_linear_oace", "fused_linear_oace_forward",
    "fused_linear_oace_backward", "fused_oace_softmax_loss", "DraftPlan", "PagePool", "append_to_cache",
    "build_block_tables", "paged_tree_afa", "paged_prefix_afa", "apply_ago_norm_rotations", "accumulate_cache_weights",
    "evict_from_cache",
]
