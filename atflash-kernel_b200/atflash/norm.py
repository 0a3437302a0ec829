"""RMS norms of the query and key heads with the RoPE rotation in the same pass
(``atf_qk_norm_rope``), for models that norm each head between projection and rotation.
``append_paged_kv_cache(k_norm=...)`` does the same to K on its way into a cache.

The reference's models have no such norms."""
from typing import Optional

import torch

from . import _ffi


def qk_norm_rope(q: torch.Tensor, k: Optional[torch.Tensor], q_weight: torch.Tensor, k_weight: Optional[torch.Tensor],
                 cos: torch.Tensor, sin: torch.Tensor, *, eps: float = 1e-6, pos_offset: int = 0,
                 positions: Optional[torch.Tensor] = None, out_layout: str = "rotate_half",
                 q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None):
    """Norm each head of q and k and rotate it: y = x w / sqrt(mean(x^2) + eps) over the 128
    elements, then RoPE of y in HF rotate_half order, in fp32 and rounded once to bf16,
    written in `out_layout` order ("rotate_half" or "sorted_pair"). Returns (q_out, k_out).

    q (B, S, Hq, 128) and k (B, S, Hk, 128), or packed tokens (T, H, 128); any strides that
    are multiples of 8 elements, so slices of one qkv projection are read in place. k and
    k_weight may be None (the append norms K itself, with ``k_norm``): k_out is then
    None. Weights: 128 bf16 or fp32, both of one type. positions: integers (S,) or (B, S), or
    (T,); default pos_offset + s; positions outside the tables are clamped into them, as
    by ``rope_pack``. q_out may be q and k_out may be k (in place); otherwise outputs overlap
    no input. A row whose squares overflow fp32 (elements over 1e18) gives 0. There is no
    backward pass."""
    return _ffi.binding().qk_norm_rope(q, k, q_weight, k_weight, cos, sin, eps, pos_offset, positions, out_layout, q_out,
                                       k_out)
