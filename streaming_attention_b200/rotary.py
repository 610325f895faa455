"""The norm of queries and keys for each head with the position rotation in the
same pass: what stands between a layer's projection and the attentions of this
package.

    y = x / sqrt(mean(x^2) + eps) * weight
    (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin),  angle = position * frequency[i]

float32 throughout, one rounding at the end; the angles are reduced in float64.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _serving as S

Tensor = torch.Tensor

__all__ = ["qk_norm_rotary", "rotary_frequencies"]


def rotary_frequencies(dim: int, *, base: float = 10000.0, device=None) -> Tensor:
    """base^(-2 i / dim) for i < dim / 2, float64: the angle per position of each
    rotated pair."""
    if dim < 0 or dim % 2:
        raise ValueError("dim must be even")
    i = torch.arange(dim // 2, dtype=torch.float64, device=device)
    return base ** (-2.0 * i / max(dim, 1))


def qk_norm_rotary(q: Tensor, k: Tensor, positions: Tensor, q_weight: Optional[Tensor], k_weight: Optional[Tensor],
                   frequencies: Tensor, *, eps: float = 1e-6, interleaved: bool = False,
                   out: Optional[Tuple[Tensor, Tensor]] = None) -> Tuple[Tensor, Tensor]:
    """Norms and rotates q [T,H,D] and k [T,Hkv,D] (any strides: slices of one
    projection) for tokens at ``positions`` (int32 [T]).  ``frequencies``
    (float64 [R]) rotates the first 2 R <= D columns of a head, as halves or,
    ``interleaved``, as neighbours.  Weights [D] in the inputs' dtype, None for
    ones.  A token of negative position is left out: its rows of a given ``out``
    pair stay as they were (``out=(q, k)`` works in place), of a new one are
    zero."""
    if q.ndim != 3 or k.ndim != 3:
        raise ValueError("q and k must be [T,H,D] and [T,Hkv,D]")
    t, heads, d = q.shape
    kt, kv_heads, kd = k.shape
    if kt != t or kd != d:
        raise ValueError("q and k must be [T,H,D] and [T,Hkv,D]")
    given = [x for x in (q_weight, k_weight) if x is not None]
    dev = S.device_of(q, k, positions, frequencies, *given)
    code = S.dtype_code(q, k, *given)
    if not 1 <= d <= S.MAX_DIM:
        raise ValueError(f"the head width must lie in [1, {S.MAX_DIM}]")
    for w in given:
        if w.ndim != 1 or w.size(0) != d:
            raise ValueError(f"q_weight and k_weight must be [{d}]")
    if heads + kv_heads == 0:
        raise ValueError("at least one head is needed")
    if frequencies.dtype != torch.float64 or frequencies.ndim != 1 or 2 * frequencies.size(0) > d:
        raise ValueError(f"frequencies must be float64 [R] with 2 R <= {d}")
    positions = S.int32(positions, (t,), "positions")
    fresh = out is None
    if fresh:
        out = q.new_empty((t, heads, d)), k.new_empty((t, kv_heads, d))
    else:
        for o, x in zip(out, (q, k)):
            if o.shape != x.shape or o.dtype != x.dtype or o.device != dev or (d > 1 and o.stride(-1) != 1):
                raise ValueError("out must match q and k, its last dimension contiguous")
            if S.repeats(o):
                raise ValueError("out must not be an expanded tensor")
    if t:
        q, k, frequencies = S.rows(q), S.rows(k), frequencies.contiguous()
        q_weight, k_weight = (None if w is None else w.contiguous() for w in (q_weight, k_weight))
        S.launch(dev, "sa_qk_norm_rotary", q.data_ptr(), k.data_ptr(), out[0].data_ptr(), out[1].data_ptr(),
                 positions.data_ptr(), S.ptr(q_weight), S.ptr(k_weight), frequencies.data_ptr(),
                 S.strides(*q.stride()[:2], *k.stride()[:2], *out[0].stride()[:2], *out[1].stride()[:2]), t, heads,
                 kv_heads, d, frequencies.size(0), float(eps), int(interleaved), int(fresh), code)
    return out[0], out[1]
