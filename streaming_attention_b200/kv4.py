"""A paged key/value cache held in 4 bits, the attention that reads it, and its
page tables.

``plan_kv_pages`` turns request lengths into page-table entries, slots and
positions on the GPU; ``Kv4Cache.append`` quantises new keys and values into
their slots, ``Kv4Cache.attend`` is the attention of each request's newest
tokens over its pages, ``Kv4Cache.read`` gives back what slots hold, and
``release_kv_pages`` returns the pages of ended requests.  Lengths, tables and
the free list stay on the device: nothing here reads them on the host, so a
decode step can be captured into a CUDA graph.

Every (token, head) row of keys and of values is held as 4-bit codes with a
scale and a least value in bfloat16 (layout in include/streaming_attention.h):

    least = bf16(min x), scale = bf16((max x - min x) / 15)
    code = clamp(round((x - least) / scale), 0, 15), value = scale * code + least
"""

from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple

import torch

from . import _serving as S

Tensor = torch.Tensor

__all__ = ["Kv4Cache", "PagePlan", "plan_kv_pages", "release_kv_pages"]

PAGE_SIZES = (16, 32, 64, 128, 256)


def _check_page_size(page_size: int) -> None:
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")


class PagePlan(NamedTuple):
    """What ``plan_kv_pages`` gives: the lengths with the new tokens, the packed
    new tokens' first rows per request [R+1], each row's position and slot (-1
    where no token stands), the page tables and how many pages stay free [1]."""
    lengths: Tensor
    offsets: Tensor
    positions: Tensor
    slots: Tensor
    tables: Tensor
    free_count: Tensor


def plan_kv_pages(lengths: Tensor, new: Tensor, tables: Tensor, free_pages: Tensor, free_count: Tensor, *,
                  page_size: int, max_tokens: Optional[int] = None, per_request: Optional[int] = None,
                  prompts: bool = False) -> PagePlan:
    """Makes room for ``new[r]`` tokens of each request behind its ``lengths[r]``
    (int32 [R]).  Pages come in request order from the end of the first
    ``free_count[0]`` entries of ``free_pages`` (int32 [F], ids below F) and are
    entered in ``tables`` (int32 [R,W], contiguous, in place; calling again with
    the same inputs enters the same).  Positions and
    slots are packed, ``max_tokens`` long, or, with ``per_request=n`` instead,
    [R*n] with n rows for each request.  Too few pages, a row of the table that is too short
    and more new tokens than rows (they count, and their pages are entered) leave
    slots at -1 and are reported by ``check_serving_status``; with ``prompts`` (and
    ``max_tokens``) so are new tokens of requests that hold some already."""
    dev = S.device_of(lengths, new, tables, free_pages, free_count)
    _check_page_size(page_size)
    if tables.ndim != 2 or tables.dtype != torch.int32 or not tables.is_contiguous():
        raise ValueError("tables must be contiguous int32 [R,W]")
    r, width = tables.shape
    lengths = S.int32(lengths, (r,), "lengths")
    new = S.int32(new, (r,), "new")
    if free_pages.ndim != 1:
        raise ValueError("free_pages must be [F]")
    free_pages = S.int32(free_pages, free_pages.shape, "free_pages")
    free_count = S.int32(free_count, (1,), "free_count")
    if (max_tokens is None) == (per_request is None):
        raise ValueError("give either max_tokens or per_request")
    if per_request is not None:
        if prompts:
            raise ValueError("prompts are packed: give max_tokens")
        if per_request <= 0:
            raise ValueError("per_request must be positive")
        max_tokens = r * per_request
    elif max_tokens < 0:
        raise ValueError("max_tokens must be non-negative")
    if max(max_tokens, free_pages.shape[0]) > 2 ** 31 - 1:
        raise ValueError("a plan takes less than 2^31 rows and pages")
    # one allocation for the outputs
    lens, offsets, positions, slots, free = lengths.new_empty(2 * r + 2 + 2 * max_tokens).split(
        (r, r + 1, max_tokens, max_tokens, 1))
    S.launch(dev, "sa_plan_kv_prompts" if prompts else "sa_plan_kv_pages", lengths.data_ptr(), new.data_ptr(),
             tables.data_ptr(), free_pages.data_ptr(), free_count.data_ptr(), r, width, free_pages.shape[0], page_size,
             max_tokens, *(() if prompts else (per_request or 0,)), lens.data_ptr(), offsets.data_ptr(), positions.data_ptr(),
             slots.data_ptr(), free.data_ptr())
    return PagePlan(lens, offsets, positions, slots, tables, free)


def release_kv_pages(lengths: Tensor, tables: Tensor, drop: Tensor, free_pages: Tensor, free_count: Tensor, *,
                     page_size: int) -> None:
    """Ends the requests with ``drop[r]`` (bool [R]): their pages go back to the
    end of the free list, their lengths to 0 and their table rows to -1, all in
    place."""
    dev = S.device_of(lengths, tables, drop, free_pages, free_count)
    _check_page_size(page_size)
    if tables.ndim != 2:
        raise ValueError("tables must be [R,W]")
    r, width = tables.shape
    if drop.dtype != torch.bool or tuple(drop.shape) != (r,):
        raise ValueError(f"drop must be bool [{r}]")
    S.int32(lengths, (r,), "lengths")
    S.int32(tables, (r, width), "tables")
    if free_pages.ndim != 1:
        raise ValueError("free_pages must be [F]")
    S.int32(free_pages, free_pages.shape, "free_pages")
    S.int32(free_count, (1,), "free_count")
    for t in (lengths, tables, free_pages, free_count):
        if not t.is_contiguous():
            raise ValueError("lengths, tables, free_pages and free_count are updated in place: they must be contiguous")
    drop = drop.contiguous()
    S.launch(dev, "sa_release_kv_pages", lengths.data_ptr(), tables.data_ptr(), drop.data_ptr(),
             free_pages.data_ptr(), free_count.data_ptr(), r, width, free_pages.shape[0], page_size)


class Kv4Cache:
    """The cache's storage.  ``Kv4Cache.empty`` makes one; the constructor takes
    the four tensors (k_codes uint8 [P,Hkv,page,Dp/2], k_params bfloat16
    [P,Hkv,page,2], v_codes uint8 [P,Hkv,page/4,Dp/2,4], v_params bfloat16
    [P,Hkv,page,2]; Dp is ``dim`` filled up to 32, 64, 128 or 256).  They are
    attributes of those names and may be replaced between calls, all four where
    the pages change; a captured call keeps those it was captured with."""

    def __init__(self, k_codes: Tensor, k_params: Tensor, v_codes: Tensor, v_params: Tensor, dim: int) -> None:
        if not 1 <= dim <= S.MAX_DIM:
            raise ValueError(f"dim must lie in [1, {S.MAX_DIM}]")
        self.k_codes, self.k_params, self.v_codes, self.v_params, self.dim = k_codes, k_params, v_codes, v_params, int(dim)
        self._bind()

    def _bind(self) -> None:
        """Checks the four tensors as they are now and keeps what the calls need of them."""
        held = k_codes, k_params, v_codes, v_params = self.k_codes, self.k_params, self.v_codes, self.v_params
        if k_codes.ndim != 4:
            raise ValueError("k_codes must be [P,Hkv,page,Dp/2]")
        pages, heads, page, half = k_codes.shape
        if page not in PAGE_SIZES:
            _check_page_size(page)
        if pages == 0 or heads == 0:
            raise ValueError("the cache needs at least one page and one head")
        if half != self.padded_dim(self.dim) // 2:
            raise ValueError(f"a row of codes of dim {self.dim} takes {self.padded_dim(self.dim) // 2} bytes, got {half}")
        device = S.device_of(k_codes, k_params, v_codes, v_params)
        params = (pages, heads, page, 2)
        for t, shape, dt, what in ((k_codes, None, torch.uint8, "k_codes"),
                                   (v_codes, (pages, heads, page // 4, half, 4), torch.uint8, "v_codes"),
                                   (k_params, params, torch.bfloat16, "k_params"),
                                   (v_params, params, torch.bfloat16, "v_params")):
            if t.dtype != dt or (shape is not None and t.shape != shape) or not t.is_contiguous():
                raise ValueError(f"{what} must be contiguous {dt} {list(shape or k_codes.shape)}")
        self.device, self.kv_heads, self.page_size, self.num_pages = device, heads, page, pages
        self._held, self._ptrs = held, (k_codes.data_ptr(), k_params.data_ptr(), v_codes.data_ptr(), v_params.data_ptr())
        self._args = (*self._ptrs, pages, heads, page, self.dim)

    def _storage(self):
        """Pointers and sizes for a call: the tensors may have been replaced, or their
        memory, since the last one."""
        k, kp, v, vp = self._held
        if (self.k_codes is not k or self.k_params is not kp or self.v_codes is not v or self.v_params is not vp or
                (k.data_ptr(), kp.data_ptr(), v.data_ptr(), vp.data_ptr()) != self._ptrs):
            self._bind()
        return self._args

    @staticmethod
    def padded_dim(dim: int) -> int:
        return max(32, 1 << (dim - 1).bit_length())

    @classmethod
    def empty(cls, num_pages: int, kv_heads: int, dim: int, *, page_size: int = 64, device=None) -> "Kv4Cache":
        """A cache of ``num_pages`` pages of ``page_size`` tokens on ``device``."""
        if not torch.cuda.is_available():
            raise ValueError("the B200 kernels need a CUDA device; none is available")
        _check_page_size(page_size)
        if not 1 <= dim <= S.MAX_DIM:
            raise ValueError(f"dim must lie in [1, {S.MAX_DIM}]")
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        half = cls.padded_dim(dim) // 2
        u8 = dict(dtype=torch.uint8, device=dev)
        b16 = dict(dtype=torch.bfloat16, device=dev)
        return cls(torch.zeros((num_pages, kv_heads, page_size, half), **u8),
                   torch.zeros((num_pages, kv_heads, page_size, 2), **b16),
                   torch.zeros((num_pages, kv_heads, page_size // 4, half, 4), **u8),
                   torch.zeros((num_pages, kv_heads, page_size, 2), **b16), dim)

    def append(self, k: Tensor, v: Tensor, slots: Tensor) -> None:
        """Quantises k and v [T,Hkv,D] into ``slots`` (int32 [T]); a negative slot
        leaves its token out, and no slot may be given twice in one call."""
        cache = self._storage()
        S.device_of(self.k_codes, k, v, slots)
        code = S.dtype_code(k, v)
        if k.ndim != 3 or k.shape[1:] != (self.kv_heads, self.dim) or v.shape != k.shape:
            raise ValueError(f"k and v must be [T,{self.kv_heads},{self.dim}]")
        slots = S.int32(slots, (k.shape[0],), "slots")
        if k.shape[0] == 0:
            return
        k, v = S.rows(k), S.rows(v)
        S.launch(self.device, "sa_kv4_append", *cache, k.data_ptr(), v.data_ptr(),
                 S.strides(*k.stride()[:2], *v.stride()[:2]), slots.data_ptr(), k.shape[0], code)

    def read(self, slots: Tensor, dtype: torch.dtype = torch.float32) -> Tuple[Tensor, Tensor]:
        """The keys and values [T,Hkv,D] that ``slots`` (int32 [T]) stand for, in
        ``dtype``; zeros for a negative slot."""
        cache = self._storage()
        S.device_of(self.k_codes, slots)
        if dtype not in S.DTYPES:
            raise ValueError(f"unsupported dtype {dtype}: float32, float16 and bfloat16 are accepted")
        if slots.ndim != 1:
            raise ValueError("slots must be [T]")
        slots = S.int32(slots, slots.shape, "slots")
        t = slots.shape[0]
        k = torch.empty((t, self.kv_heads, self.dim), device=self.device, dtype=dtype)
        v = torch.empty((t, self.kv_heads, self.dim), device=self.device, dtype=dtype)
        if t:
            S.launch(self.device, "sa_kv4_read", *cache, k.data_ptr(), v.data_ptr(), slots.data_ptr(), t,
                     S.DTYPES[dtype])
        return k, v

    def attend(self, q: Tensor, tables: Tensor, lengths: Tensor, *, window: Optional[int] = None, sinks: int = 0,
               scale: Optional[float] = None) -> Tensor:
        """Attention of each request's newest tokens over its cached ones.

        q [R,H,D] (one token each) or [R,N,H,D] (the last N of each request);
        ``tables`` int32 [R,W], ``lengths`` int32 [R] count the new tokens, which
        are appended before.  Query i of N stands at lengths[r] - N + i and sees
        as in ``sliding_window_attention``; a query that sees nothing (a request
        of length 0, or shorter than N) gives zeros.  Returns q's shape and dtype."""
        cache = self._storage()
        S.device_of(self.k_codes, q, tables, lengths)
        code = S.dtype_code(q)
        w, s = S.check_window(window, sinks)
        if q.ndim not in (3, 4):
            raise ValueError("q must be [R,H,D] or [R,N,H,D]")
        q4 = q[:, None] if q.ndim == 3 else q
        r, n, heads, d = q4.shape
        if d != self.dim or heads == 0 or heads % self.kv_heads:
            raise ValueError(f"q must have head width {self.dim} and a multiple of {self.kv_heads} heads")
        if tables.ndim != 2 or tables.shape[0] != r:
            raise ValueError(f"tables must be [{r},W]")
        tables = S.int32(tables, tables.shape, "tables")
        lengths = S.int32(lengths, (r,), "lengths")
        out = torch.empty((r, n, heads, d), device=self.device, dtype=q.dtype)
        if out.numel():
            q4 = S.rows(q4)
            S.launch(self.device, "sa_kv4_attend", *cache, q4.data_ptr(), out.data_ptr(),
                     S.strides(*q4.stride()[:3]), tables.data_ptr(), lengths.data_ptr(), r, n, heads, tables.shape[1],
                     w, s, float(1.0 / math.sqrt(d) if scale is None else scale), code)
        return out[:, 0] if q.ndim == 3 else out
