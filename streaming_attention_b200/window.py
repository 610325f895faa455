"""Exact attention with a sliding window and a few first tokens that stay
visible ("sinks"), beside the framework's exact causal attention
(``triton_flash_causal_attention``): bounded work per query, grouped heads,
16-bit tensor cores, continued prompts (fewer queries than keys) and ragged
batches.  Forward only, as everywhere in this package.

    out_i = sum_j softmax_j(scale q_i.k_j) v_j   over the visible keys
    j <= p and (j > p - window or j < sinks),    p = m - n + i

A query that sees nothing gives zeros.  Scores, softmax and sums are float32;
with 16-bit inputs the probabilities are rounded to the inputs' type before
their product with v (the operand type of the tensor cores).
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _lib
from . import _serving as S

Tensor = torch.Tensor

__all__ = ["sliding_window_attention", "sliding_window_attention_packed"]


def _scale(scale: Optional[float], dim: int) -> float:
    return float(1.0 / math.sqrt(dim) if scale is None else scale)


def _check_dims(q: Tensor, k: Tensor, v: Tensor) -> None:
    if q.shape[-1] != k.shape[-1]:
        raise ValueError(f"q and k must have the same head width, got {q.shape[-1]} and {k.shape[-1]}")
    if not 1 <= q.shape[-1] <= S.MAX_DIM or not 1 <= v.shape[-1] <= S.MAX_DIM:
        raise ValueError(f"head widths must lie in [1, {S.MAX_DIM}]")


def _check_heads(heads: int, kv_heads: int) -> None:
    if kv_heads == 0 or heads % kv_heads != 0:
        raise ValueError(f"the query heads ({heads}) must be a multiple of the key heads ({kv_heads})")


def _workspace_size(*sizes: int) -> int:
    nbytes = ctypes.c_size_t(0)
    _lib.check(_lib.load().sa_window_attention_workspace_size(*sizes, ctypes.byref(nbytes)), "window workspace size")
    return nbytes.value


def _on_borders(t: Tensor) -> Tensor:
    """t, or a copy of it, as the kernels read it: a contiguous last dimension
    and, for 16-bit types of widths the tensor cores take, rows that start on
    16-byte borders (TMA) and are no repeats of one another."""
    d = t.shape[-1]
    if d % 8 == 0 and t.is_contiguous() and t.data_ptr() % 16 == 0:   # the usual tensor, without a look at each stride
        return t
    t = S.rows(t)
    if t.dtype == torch.float32 or d > 128:
        return t
    if t.data_ptr() % 16 == 0 and all(st > 0 and st % 8 == 0 or n <= 1 for n, st in zip(t.shape, t.stride()[:-1])):
        return t
    wide = torch.empty(t.shape[:-1] + ((d + 7) // 8 * 8,), device=t.device, dtype=t.dtype)[..., :d]
    return wide.copy_(t.detach())


def sliding_window_attention(q: Tensor, k: Tensor, v: Tensor, *, window: Optional[int], sinks: int = 0,
                             scale: Optional[float] = None) -> Tensor:
    """Windowed attention of [N,D] or [B,H,N,D] queries over [M,D] or [B,Hkv,M,D]
    keys and [.., M, Dv] values, M >= N: the queries stand at the last N of the
    M positions.  ``window=None`` hides nothing but later keys.  H is a multiple
    of Hkv (query head h reads key head h // (H / Hkv)).  float32, float16 or
    bfloat16, any strides; the result is contiguous in the inputs' dtype."""
    dev = S.device_of(q, k, v)
    if not q.ndim == k.ndim == v.ndim or q.ndim not in (2, 4):
        raise ValueError("q/k/v must be [N,D] or [B,H,N,D]")
    w, s = S.check_window(window, sinks)
    code = S.dtype_code(q, k, v)
    _check_dims(q, k, v)
    if k.shape[:-1] != v.shape[:-1]:
        raise ValueError("v must match k in every dimension but the last")
    single = q.ndim == 2
    if single:
        q, k, v = q[None, None], k[None, None], v[None, None]
    b, heads, n, d = q.shape
    kv_heads, m, dv = k.shape[1], k.shape[2], v.shape[3]
    if k.shape[0] != b:
        raise ValueError("q, k and v must have the same batch size")
    if m < n:
        raise ValueError(f"fewer keys ({m}) than queries ({n})")
    out = q.new_empty((b, heads, n, dv))
    if out.numel():
        _check_heads(heads, kv_heads)
        ws = None
        # 16 bits: 48 tiles of 64 keys and more may be split, longer chains folded
        if q.dtype == torch.float32 or m > 3008:
            size = _workspace_size(b, heads, kv_heads, n, m, d, dv, w, s, code)
            if size:
                ws = torch.empty(size, device=dev, dtype=torch.uint8)
                if q.dtype == torch.float32:
                    q, k, v = (t.detach().contiguous() for t in (q, k, v))
        q, k, v = _on_borders(q), _on_borders(k), _on_borders(v)
        S.launch(dev, "sa_window_attention", q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                 S.strides(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *out.stride()[:3]), b, heads, kv_heads,
                 n, m, d, dv, w, s, _scale(scale, d), code, None, None, 0,
                 None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel())
    return out[0, 0] if single else out


def sliding_window_attention_packed(q: Tensor, k: Tensor, v: Tensor, cu_q: Tensor, cu_k: Tensor, *,
                                    window: Optional[int], sinks: int = 0, scale: Optional[float] = None,
                                    out: Optional[Tensor] = None) -> Tensor:
    """Windowed attention of a ragged batch packed along the rows: q [T,H,D], k
    [S,Hkv,D], v [S,Hkv,Dv]; ``cu_q`` and ``cu_k`` (int32 [R+1], on the device)
    are the requests' first rows, so that request r has rows cu_q[r]..cu_q[r+1]
    of q and cu_k[r]..cu_k[r+1] of k and v, its queries at the last of its
    positions.  No length is read on the host: a request whose offsets are out of
    order or range is skipped, and reported by ``check_serving_status``.  Rows of
    no request (behind cu_q[R]) and of a skipped one are left as they were in
    ``out`` ([T,H,Dv]); in a new one they are zero."""
    dev = S.device_of(q, k, v, cu_q, cu_k)
    if not q.ndim == k.ndim == v.ndim == 3:
        raise ValueError("q, k and v must be [T,H,D], [S,Hkv,D], [S,Hkv,Dv]")
    w, s = S.check_window(window, sinks)
    code = S.dtype_code(q, k, v)
    _check_dims(q, k, v)
    if k.shape[:-1] != v.shape[:-1]:
        raise ValueError("v must match k in every dimension but the last")
    t, heads, d = q.shape
    rows, kv_heads, dv = v.shape
    if cu_q.ndim != 1 or cu_q.shape[0] < 1:
        raise ValueError("cu_q must be [R+1]")
    cu_q = S.int32(cu_q, cu_q.shape, "cu_q")
    cu_k = S.int32(cu_k, cu_q.shape, "cu_k")
    fresh = out is None
    if fresh:
        out = q.new_empty((t, heads, dv)) if cu_q.size(0) > 1 else q.new_zeros((t, heads, dv))
    elif tuple(out.shape) != (t, heads, dv) or out.dtype != q.dtype or out.device != dev or (dv > 1 and out.stride(-1) != 1):
        raise ValueError(f"out must be [{t},{heads},{dv}] like q, its last dimension contiguous")
    elif S.repeats(out):
        raise ValueError("out must not be an expanded tensor")
    if out.numel():
        _check_heads(heads, kv_heads)
        ws, size = None, 0
        if code != _lib.REP_DTYPES["float32"] and rows > 32000 and (w == 0 or w + s > 31900):   # long chains are folded
            size = _workspace_size(1, heads, kv_heads, rows, rows, d, dv, w, s, code)
            ws = torch.empty(size, device=dev, dtype=torch.uint8) if size else None
        q, k, v = _on_borders(q), _on_borders(k), _on_borders(v)
        S.launch(dev, "sa_window_attention", q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                 S.strides(0, q.stride(1), q.stride(0), 0, k.stride(1), k.stride(0), 0, v.stride(1), v.stride(0), 0,
                           out.stride(1), out.stride(0)), cu_q.shape[0] - 1, heads, kv_heads, t, rows, d, dv, w, s,
                 _scale(scale, d), code, cu_q.data_ptr(), cu_k.data_ptr(), int(fresh), S.ptr(ws), size)
    return out
