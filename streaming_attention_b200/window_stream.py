"""Streaming attention of a batch of requests over a 4-bit cache with a sliding
window and first tokens that stay visible: the batched, bounded-window
counterpart of ``ArticleStreamingAttention``.

One object is one layer's attention: ``prefill`` takes the prompts of new
requests (packed, ragged), ``decode`` the next tokens of the batch.  Both norm
and rotate queries and keys, make room in the cache, write the new keys and
values to it and attend: a prompt over its own keys at full precision, a decode
step over the cache.  The window bounds the work of a step, not the cache: a
request keeps the pages of all its tokens until it is released.  Lengths, page
tables and the free list live on the device at fixed addresses, so ``decode`` can
be captured into a CUDA graph.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _serving as S
from .kv4 import Kv4Cache, PagePlan, plan_kv_pages, release_kv_pages
from .rotary import qk_norm_rotary, rotary_frequencies
from .window import sliding_window_attention_packed

Tensor = torch.Tensor

__all__ = ["StreamingWindowAttention"]


class StreamingWindowAttention:
    """Attention layer state for up to ``max_requests`` requests of up to
    ``max_length`` tokens each.

    ``q_weight`` / ``k_weight`` [dim] are the norms' weights (None: ones),
    ``frequencies`` the rotation's (float64, default ``rotary_frequencies(dim)``
    for even ``dim``).  ``num_pages`` defaults to room for every request at its
    longest."""

    def __init__(self, heads: int, kv_heads: int, dim: int, *, max_requests: int, max_length: int,
                 window: Optional[int] = None, sinks: int = 0, scale: Optional[float] = None,
                 q_weight: Optional[Tensor] = None, k_weight: Optional[Tensor] = None,
                 frequencies: Optional[Tensor] = None, eps: float = 1e-6, interleaved: bool = False,
                 page_size: int = 64, num_pages: Optional[int] = None, device=None) -> None:
        if heads <= 0 or kv_heads <= 0 or heads % kv_heads:
            raise ValueError("the query heads must be a positive multiple of the key heads")
        if max_requests <= 0 or max_length <= 0:
            raise ValueError("max_requests and max_length must be positive")
        S.check_window(window, sinks)
        width = -(-max_length // page_size) if page_size > 0 else 0
        pages = max_requests * width if num_pages is None else num_pages
        self.cache = Kv4Cache.empty(pages, kv_heads, dim, page_size=page_size, device=device)
        dev = self.cache.device
        self.device, self.heads, self.kv_heads, self.dim = dev, heads, kv_heads, dim
        self.window, self.sinks, self.scale, self.eps, self.interleaved = window, sinks, scale, eps, interleaved
        self.q_weight, self.k_weight = q_weight, k_weight
        self.frequencies = rotary_frequencies(dim - dim % 2, device=dev) if frequencies is None else frequencies
        i32 = dict(device=dev, dtype=torch.int32)
        self.lengths = torch.zeros(max_requests, **i32)
        self.tables = torch.full((max_requests, width), -1, **i32)
        self.free_pages = torch.arange(pages - 1, -1, -1, **i32)   # page 0 is taken first
        self.free_count = torch.full((1,), pages, **i32)

    def _step(self, q: Tensor, k: Tensor, v: Tensor, new: Tensor, **rows):
        """Plan, norm and rotation, append; returns the plan and the rotated q, k."""
        t = q.shape[0]
        if tuple(q.shape) != (t, self.heads, self.dim) or tuple(k.shape) != (t, self.kv_heads, self.dim) or v.shape != k.shape:
            raise ValueError(f"q, k, v must be [T,{self.heads},{self.dim}], [T,{self.kv_heads},{self.dim}] (twice)")
        S.dtype_code(q, k, v)
        S.device_of(self.lengths, q, k, v, new)
        plan: PagePlan = plan_kv_pages(self.lengths, new, self.tables, self.free_pages, self.free_count,
                                       page_size=self.cache.page_size, **rows)
        q, k = qk_norm_rotary(q, k, plan.positions, self.q_weight, self.k_weight, self.frequencies, eps=self.eps,
                              interleaved=self.interleaved)
        self.cache.append(k, v, plan.slots)
        self.lengths.copy_(plan.lengths)
        self.free_count.copy_(plan.free_count)
        return plan, q, k

    def prefill(self, q: Tensor, k: Tensor, v: Tensor, new: Tensor) -> Tensor:
        """Prompts of requests that hold nothing yet: ``new`` (int32
        [max_requests]) tokens of each, packed in request order in q [T,H,D], k
        and v [T,Hkv,D]; T may be larger than their sum (rows behind stay zero).
        Requests with new[r] = 0 are left alone, whatever they hold; new tokens of
        one that holds some would not see them, and are reported by
        ``check_serving_status``."""
        plan, q, k = self._step(q, k, v, new, max_tokens=q.shape[0], prompts=True)
        return sliding_window_attention_packed(q, k, v, plan.offsets, plan.offsets, window=self.window,
                                               sinks=self.sinks, scale=self.scale)

    def decode(self, q: Tensor, k: Tensor, v: Tensor) -> Tensor:
        """The next token of every request: q [max_requests,H,D], k and v
        [max_requests,Hkv,D], one row for each request; a request that holds
        nothing is idle (its row is not looked at, its output is zero)."""
        if q.shape[0] != self.lengths.shape[0]:
            raise ValueError(f"decode takes one row for each of the {self.lengths.shape[0]} requests")
        _, q, _ = self._step(q, k, v, (self.lengths > 0).to(torch.int32), per_request=1)
        return self.cache.attend(q, self.tables, self.lengths, window=self.window, sinks=self.sinks, scale=self.scale)

    def release(self, drop: Tensor) -> None:
        """Ends the requests with drop[r] (bool [max_requests])."""
        release_kv_pages(self.lengths, self.tables, drop, self.free_pages, self.free_count,
                         page_size=self.cache.page_size)
