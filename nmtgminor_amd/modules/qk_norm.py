"""Norms of queries and keys for each head with the rotation to their positions, in one pass.

    qk_norm_rotary_func(q [T, B, H, D], k [T, B, H_kv, D], q_weight, k_weight, cos, sin, positions, eps) -> (q, k) like the inputs

Every head's row x becomes y = x / sqrt(mean(x^2) + eps) * weight, then y cos + rotate_half(y) sin, where rotate_half(y) =
(-y[D / 2:], y[:D / 2]) as in modules/rotary.py and cos and sin are the rows of two tables at the row's position. Differentiable in q, k
and the weights. fp16 / bf16, head dimension 64 or 128; torch.jit.trace is refused.
"""
import torch

from .. import _lib as L
from ._autocast import cast_if_autocast_enabled, no_autocast


def qk_norm_rotary_func(q, k, q_weight, k_weight, cos, sin, positions=None, eps=1e-6):
    """q and k may be slots of one projection (any strides with a contiguous D that are multiples of 8). Weights [D], fp32 or of the
    rows' type, or None for both (under autocast weights and tables of 16 bits take its type with the rows). cos, sin: [positions, D] or [positions, 1, D], fp32 or of the rows' type. positions: None (row t of
    the tables for position t), an int (of the first row), integers [B] on the device (of every sequence's first row: a decoder's
    lengths) or [T, B] (of every row). An int that leads out of the tables is an error, positions on the device are clamped to them."""
    L.refuse_tracing("qk_norm_rotary")
    start = 0
    if positions is not None and not isinstance(positions, torch.Tensor):
        positions, start = None, int(positions)
    if not torch.is_autocast_enabled():
        return L.host().qk_norm_rotary(q, k, q_weight, k_weight, cos, sin, positions, start, eps)
    q, k = cast_if_autocast_enabled(q, k)
    # (those in 32 bits stay so)
    q_weight, k_weight, cos, sin = (x.to(q.dtype) if x is not None and x.dtype in (torch.float16, torch.bfloat16) else x for x in (q_weight, k_weight, cos, sin))
    with no_autocast():
        return L.host().qk_norm_rotary(q, k, q_weight, k_weight, cos, sin, positions, start, eps)
