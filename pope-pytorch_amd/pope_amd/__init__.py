"""pope_amd: PoPE attention for AMD Instinct MI355X (gfx950).

Drop-in for the public API of lucidrains/PoPE-pytorch (``PoPE_pytorch/__init__.py:1-11``):
``PoPE``, ``apply_pope_to_qk``, ``compute_attn_similarity``, ``flash_attn_with_pope``,
``AxialPoPE``; for serving, a paged cache and the attention over it (``paged.py``); linear attention with a decay for
each head, for training and serving (``linear.py``).  GPU tensors run hand-written HIP kernels (libpope_hip.so, C ABI in
include/pope_abi.h) registered as ``torch.library`` ops under the ``pope_amd``
namespace.
"""
from .pope import PoPE, PolarEmbedReturn, apply_pope_to_qk
from .pope_nd import AxialPoPE
from .paged import PagedPoPECache, paged_cache_read, paged_cache_write, paged_flash_attn_with_pope
from .linear import gated_head_norm, linear_attn_step_with_pope, linear_attn_with_pope
from .attention import compute_attn_similarity, compute_attn_similarity_non_fused, flash_attn_with_pope

__all__ = [
    "PoPE", "PolarEmbedReturn", "apply_pope_to_qk", "AxialPoPE",
    "compute_attn_similarity", "compute_attn_similarity_non_fused", "flash_attn_with_pope",
    "PagedPoPECache", "paged_cache_write", "paged_cache_read", "paged_flash_attn_with_pope",
    "linear_attn_with_pope", "linear_attn_step_with_pope", "gated_head_norm",
]
