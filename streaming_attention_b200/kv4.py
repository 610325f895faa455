"""A paged key/value cache held in 4 bits, the attention that reads it, and its
page tables.

``plan_kv_pages`` turns request lengths into page-table entries, slots and
positions on the GPU; ``Kv4Cache.append`` quantises new keys and values into
their slots, ``Kv4Cache.attend`` is the attention of each request's newest
tokens over its pages, ``Kv4Cache.read`` gives back what slots hold, and
``release_kv_pages`` returns the pages of ended requests.  Lengths, tables and
the free list stay on the device: nothing here reads them on the host, so a
decode step can be captured into a CUDA graph.

For long requests: ``attend_shared`` computes a prefix that all requests share
once for all; ``update_page_bounds`` / ``select_pages`` / ``attend_pages`` read, for each
query, only the pages whose keys may matter most to it; ``attend(weights=...)`` adds up
what weight each token had, and ``evict`` drops the tokens of little weight.

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
        shape = k_codes.shape
        if len(shape) != 4:
            raise ValueError("k_codes must be [P,Hkv,page,Dp/2]")
        pages, heads, page, half = shape
        if page not in PAGE_SIZES:
            _check_page_size(page)
        if pages == 0 or heads == 0:
            raise ValueError("the cache needs at least one page and one head")
        if half != self.padded_dim(self.dim) // 2:
            raise ValueError(f"a row of codes of dim {self.dim} takes {self.padded_dim(self.dim) // 2} bytes, got {half}")
        device = S.device_of(k_codes, k_params, v_codes, v_params)
        params = (pages, heads, page, 2)
        for t, want, dt, what in ((k_codes, shape, torch.uint8, "k_codes"),
                                  (v_codes, (pages, heads, page // 4, half, 4), torch.uint8, "v_codes"),
                                  (k_params, params, torch.bfloat16, "k_params"),
                                  (v_params, params, torch.bfloat16, "v_params")):
            if t.dtype != dt or t.shape != want or not t.is_contiguous():
                raise ValueError(f"{what} must be contiguous {dt} {list(want)}")
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

    def _queries(self, q: Tensor, tables: Tensor, lengths: Tensor):
        """q [R,H,D] or [R,N,H,D], tables and lengths as the kernels read them: pointers and
        sizes for a call (q, its strides, tables, lengths; R, N, H, W; the element type's code), and
        the tensors that they are of."""
        shape = q.shape
        if len(shape) == 4:
            r, n, heads, d = shape
        elif len(shape) == 3:
            r, heads, d = shape
            n = 1
        else:
            raise ValueError("q must be [R,H,D] or [R,N,H,D]")
        code = S.DTYPES.get(q.dtype)
        if code is None:
            code = S.dtype_code(q)
        if d != self.dim or heads == 0 or heads % self.kv_heads:
            raise ValueError(f"q must have head width {self.dim} and a multiple of {self.kv_heads} heads")
        table_shape = tables.shape
        if len(table_shape) != 2 or table_shape[0] != r:
            raise ValueError(f"tables must be [{r},W]")
        if max(r, n, heads, table_shape[1]) >= 1 << 31:
            S.below_2_31(R=r, N=n, H=heads, W=table_shape[1])
        tables = S.int32(tables, table_shape, "tables")
        lengths = S.int32(lengths, (r,), "lengths")
        st = q.stride()
        if st[-1] != 1 and d > 1:
            q = q.detach().contiguous()
            st = q.stride()
        st = S.strides(st[0], st[1], st[2]) if len(shape) == 4 else S.strides(st[0], 0, st[1])
        return ((q.data_ptr(), st, tables.data_ptr(), lengths.data_ptr()), (r, n, heads, table_shape[1]), code, (q, tables, lengths))

    def _scale(self, scale: Optional[float]) -> float:
        return float(1.0 / math.sqrt(self.dim) if scale is None else scale)

    def attend(self, q: Tensor, tables: Tensor, lengths: Tensor, *, window: Optional[int] = None, sinks: int = 0,
               scale: Optional[float] = None, weights: Optional[Tensor] = None) -> Tensor:
        """Attention of each request's newest tokens over its cached ones.

        q [R,H,D] (one token each) or [R,N,H,D] (the last N of each request);
        ``tables`` int32 [R,W], ``lengths`` int32 [R] count the new tokens, which
        are appended before.  Query i of N stands at lengths[r] - N + i and sees
        as in ``sliding_window_attention``; a query that sees nothing (a request
        of length 0, or shorter than N) gives zeros.  Returns q's shape and dtype.

        ``weights`` (``token_weights()``, float32 [P,Hkv,page]) is added to, in place: at each
        token's slot the softmax weight it had, summed over the N queries and the
        heads that read the key head.  No page may then stand in two requests' tables; the call
        takes a workspace of 4 bytes for each query row and token that ``tables`` (and the window) allow."""
        cache = self._storage()
        if weights is None:
            S.device_of(self.k_codes, q, tables, lengths)
        else:
            S.device_of(self.k_codes, q, tables, lengths, weights)
            self._check_weights(weights)
        w, s = S.check_window(window, sinks)
        (qp, st, tp, lp), (r, n, heads, width), code, held = self._queries(q, tables, lengths)
        out = q.new_empty(q.shape)
        if r and n:
            if weights is None:
                S.launch(self.device, "sa_kv4_attend", *cache, qp, out.data_ptr(), st, tp, lp, r, n, heads, width, w, s,
                         self._scale(scale), code)
            else:
                ws = S.workspace(self.device, "sa_kv4_attend_weigh_workspace_size", self.kv_heads, self.page_size, r, n,
                                 heads, width, w, s)
                S.launch(self.device, "sa_kv4_attend_weigh", *cache, qp, out.data_ptr(), st, tp, lp, r, n, heads, width, w, s,
                         self._scale(scale), code, weights.data_ptr(), ws.data_ptr(), ws.numel())
        return out

    def attend_shared(self, q: Tensor, prefix_table: Tensor, prefix_length: Tensor, tables: Tensor, lengths: Tensor, *,
                      window: Optional[int] = None, sinks: int = 0, scale: Optional[float] = None) -> Tensor:
        """``attend`` of a batch whose requests share a prefix, which is read and computed
        once for all: request r's tokens are those of the prefix (``prefix_length`` int32 [1]
        in pages ``prefix_table`` int32 [W0]) and behind them its own (``lengths[r]``
        in pages ``tables[r]``).  The queries are the last N of its own tokens; one that it does
        not have (a request of length 0, or shorter than N) gives zeros.  Positions, ``window`` and
        ``sinks`` count from the prefix's first token.

        16-bit queries of width up to 128 and more than 32 rows a key head go over the prefix with
        probabilities and values rounded to float16 (2^-11 of each).  Where one visible token's
        keys are 2^-16 of the largest of its part, or its values 2^-13, and not zero, float32
        takes over, up to 200 times slower.  The call takes a workspace of 4 bytes for each row and
        padded column, times the parts the prefix is cut into (at least one for each 32768 tokens)."""
        cache = self._storage()
        S.device_of(self.k_codes, q, prefix_table, prefix_length, tables, lengths)
        w, s = S.check_window(window, sinks)
        (qp, st, tp, lp), (r, n, heads, width), code, held = self._queries(q, tables, lengths)
        prefix_shape = prefix_table.shape
        if len(prefix_shape) != 1:
            raise ValueError("prefix_table must be [W0]")
        S.below_2_31(W0=prefix_shape[0])
        prefix_table = S.int32(prefix_table, prefix_shape, "prefix_table")
        prefix_length = S.int32(prefix_length, (1,), "prefix_length")
        out = q.new_empty(q.shape)
        if r and n:
            ws = S.workspace(self.device, "sa_kv4_attend_shared_workspace_size", self.kv_heads, self.page_size, self.dim, r, n,
                             heads, prefix_shape[0], w, s, code)
            S.launch(self.device, "sa_kv4_attend_shared", *cache, qp, out.data_ptr(), st, prefix_table.data_ptr(),
                     prefix_length.data_ptr(), prefix_shape[0], tp, lp, r, n, heads, width, w, s, self._scale(scale), code,
                     ws.data_ptr(), ws.numel())
        return out

    def attend_pages(self, q: Tensor, tables: Tensor, lengths: Tensor, pages: Tensor, *,
                     scale: Optional[float] = None) -> Tensor:
        """``attend`` over chosen pages alone: ``pages`` int32 [R,Hkv,K] ([R,N,Hkv,K] for q
        [R,N,H,D]) lists for each query and key head rows of the request's table, in
        ascending order, -1 behind (as ``select_pages`` gives them).  A query sees the tokens
        up to its own that stand in them."""
        cache = self._storage()
        S.device_of(self.k_codes, q, tables, lengths, pages)
        (qp, st, tp, lp), (r, n, heads, width), code, held = self._queries(q, tables, lengths)
        lead = (r, self.kv_heads) if q.ndim == 3 else (r, n, self.kv_heads)
        if pages.ndim != len(lead) + 1:
            raise ValueError(f"pages must be {[*lead, 'K']}")
        count = pages.shape[-1]
        S.below_2_31(K=count)
        pages = S.int32(pages, (*lead, count), "pages")
        out = q.new_empty(q.shape)
        if r and n:
            S.launch(self.device, "sa_kv4_attend_pages", *cache, qp, out.data_ptr(), st, tp, lp, pages.data_ptr(), count, r, n,
                     heads, width, self._scale(scale), code)
        return out

    def page_bounds(self) -> Tensor:
        """Room for the bounds of every page's keys, bfloat16 [P,Hkv,2,Dp], zeros."""
        self._storage()
        shape = (self.num_pages, self.kv_heads, 2, self.padded_dim(self.dim))
        return torch.zeros(shape, dtype=torch.bfloat16, device=self.device)

    def _check_bounds(self, bounds: Tensor) -> None:
        shape = (self.num_pages, self.kv_heads, 2, self.padded_dim(self.dim))
        if bounds.dtype != torch.bfloat16 or bounds.shape != shape or not bounds.is_contiguous():
            raise ValueError(f"bounds must be contiguous bfloat16 {list(shape)}")

    def update_page_bounds(self, bounds: Tensor, tables: Tensor, lengths: Tensor, new: Tensor) -> None:
        """Writes to ``bounds`` the least and the largest value of each column of the keys
        that the pages of each request's newest ``new[r]`` (int32 [R]) tokens hold;
        ``lengths`` counts them, as after ``append``.  Other pages' bounds stay.  A page in two
        requests' tables holds the same tokens of both."""
        cache = self._storage()
        S.device_of(self.k_codes, bounds, tables, lengths, new)
        self._check_bounds(bounds)
        if tables.ndim != 2:
            raise ValueError("tables must be [R,W]")
        S.below_2_31(R=tables.shape[0], W=tables.shape[1])
        tables = S.int32(tables, tables.shape, "tables")
        r, width = tables.shape
        lengths = S.int32(lengths, (r,), "lengths")
        new = S.int32(new, (r,), "new")
        if r and width:
            S.launch(self.device, "sa_kv4_page_bounds", *cache, bounds.data_ptr(), tables.data_ptr(), lengths.data_ptr(),
                     new.data_ptr(), r, width)

    def select_pages(self, q: Tensor, bounds: Tensor, tables: Tensor, lengths: Tensor, *, count: int, first: int = 1,
                     last: int = 1) -> Tensor:
        """The ``count`` pages each query should read, int32 [R,Hkv,count] ([R,N,Hkv,count] for
        q [R,N,H,D]): rows of the request's table, ascending, -1 behind.  Of the pages up
        to the query's own the ``first`` first and the ``last`` last are always among them; of
        those between, the ones of the largest

            score = sum over the heads of a key head, columns c, of max(q_c low_c, q_c high_c)

        with the page's ``bounds`` (of equal scores the lowest page; NaN, which 0 times an infinite
        bound gives, is the largest)."""
        self._storage()
        S.device_of(self.k_codes, q, bounds, tables, lengths)
        self._check_bounds(bounds)
        (qp, st, tp, lp), (r, n, heads, width), code, held = self._queries(q, tables, lengths)
        count, first, last = S.whole(count, "count"), S.whole(first, "first"), S.whole(last, "last")
        if not 0 <= count <= 1 << 30:
            raise ValueError("count must lie in [0, 2^30]")
        if first < 0 or last < 0 or first + last > count:
            raise ValueError("first and last must be non-negative, and no more than count together")
        out = lengths.new_empty((r, self.kv_heads, count) if q.ndim == 3 else (r, n, self.kv_heads, count))
        if r and n and count:
            S.launch(self.device, "sa_kv4_select_pages", bounds.data_ptr(), self.num_pages, self.kv_heads, self.page_size,
                     self.dim, qp, st, tp, lp, r, n, heads, width, count, first, last, code, out.data_ptr())
        return out

    def token_weights(self) -> Tensor:
        """Room for the weight of every token, float32 [P,Hkv,page], zeros."""
        self._storage()
        return torch.zeros((self.num_pages, self.kv_heads, self.page_size), dtype=torch.float32, device=self.device)

    def _check_weights(self, weights: Tensor) -> None:
        shape = (self.num_pages, self.kv_heads, self.page_size)
        if weights.dtype != torch.float32 or weights.shape != shape or not weights.is_contiguous():
            raise ValueError(f"weights must be contiguous float32 {list(shape)}")

    def reset_weights(self, weights: Tensor, slots: Tensor) -> None:
        """Zeros for the weights of ``slots`` (int32 [T], negative: none): what new tokens start
        from, where others stood before."""
        self._storage()
        S.device_of(self.k_codes, weights, slots)
        self._check_weights(weights)
        if slots.ndim != 1:
            raise ValueError("slots must be [T]")
        slots = S.int32(slots, slots.shape, "slots")
        if slots.shape[0]:
            S.launch(self.device, "sa_kv4_reset_weights", weights.data_ptr(), self.num_pages, self.kv_heads, self.page_size,
                     slots.data_ptr(), slots.shape[0])

    def evict(self, weights: Tensor, lengths: Tensor, tables: Tensor, free_pages: Tensor, free_count: Tensor, *, keep: int,
              limit: Optional[int] = None, first: int = 0, last: int = 0) -> Tuple[Tensor, Tensor]:
        """Drops tokens of little weight, in place: a request of more than ``limit`` tokens
        (default ``keep``) keeps ``keep`` of each key head -- its ``first`` first ones, its ``last``
        newest ones and, between, those of the largest ``weights`` (of equal ones the
        lowest; NaN is the largest) -- moved up in order, with their weights, to its first slots.  Its
        length becomes ``keep``; the pages behind go to the end of the free list; the weights
        of the slots behind become zero.

        Returns which tokens each head kept (int32 [R,Hkv,keep]; of a request that was not
        over 0, 1, .. and -1 behind its last) and how many a request lost (int32 [R]): its next
        token's position is its length plus all it ever lost.  Heads keep tokens of their
        own, so ``window`` and ``sinks`` count what is held, and bounds of its pages are to be
        updated as a whole.  No page may stand in two requests' tables.  Up to 16384 requests a call, of tables of
        up to 2^30 tokens."""
        cache = self._storage()
        S.device_of(self.k_codes, weights, lengths, tables, free_pages, free_count)
        self._check_weights(weights)
        keep, first, last = S.whole(keep, "keep"), S.whole(first, "first"), S.whole(last, "last")
        limit = keep if limit is None else S.whole(limit, "limit")
        if not 1 <= keep <= limit <= 2 ** 31 - 1:
            raise ValueError("keep must be positive, and limit no less")
        if first < 0 or last < 0 or first + last > keep:
            raise ValueError("first and last must be non-negative, and no more than keep together")
        if tables.ndim != 2:
            raise ValueError("tables must be [R,W]")
        if free_pages.ndim != 1:
            raise ValueError("free_pages must be [F]")
        r, width = tables.shape
        S.below_2_31(R=r, W=width, F=free_pages.shape[0])
        S.int32(lengths, (r,), "lengths")
        S.int32(tables, (r, width), "tables")
        S.int32(free_pages, free_pages.shape, "free_pages")
        S.int32(free_count, (1,), "free_count")
        for t in (lengths, tables, free_pages, free_count):
            if not t.is_contiguous():
                raise ValueError("lengths, tables, free_pages and free_count are updated in place: they must be contiguous")
        kept, dropped = lengths.new_empty((r, self.kv_heads, keep)), lengths.new_empty((r,))
        if r:
            S.launch(self.device, "sa_kv4_evict", *cache, weights.data_ptr(), lengths.data_ptr(), tables.data_ptr(),
                     free_pages.data_ptr(), free_count.data_ptr(), r, width, free_pages.shape[0], keep, limit, first, last,
                     kept.data_ptr(), dropped.data_ptr())
        return kept, dropped
