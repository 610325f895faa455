"""Selection with bounds that are infinite: of keys that pass float32 or bfloat16."""

import math

import pytest
import torch

import long_cache_ref as L
import serving_ref as R
import streaming_attention_b200 as sa
from test_long_cache_gpu import BF16, F16, F32, TYPES, _i32, _queries

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return torch.device("cuda:0")


def _check(cache, bounds, q, pages, count, first, last):
    """One request of `pages` pages in order: q [1,N,H,D]."""
    n, heads, d, h = q.shape[1], q.shape[2], q.shape[3], cache.kv_heads
    tables = torch.arange(pages, dtype=torch.int32, device=q.device)[None]
    length = pages * cache.page_size
    got = cache.select_pages(q, bounds, tables, _i32([length], q.device), count=count, first=first, last=last)
    b, qc, per = bounds.cpu().double()[..., :d], q.cpu().double(), heads // h
    for i in range(n):
        for j in range(h):
            want = L.select(qc[0, i, j * per:(j + 1) * per], b[:, j, 0], b[:, j, 1], pages, count, first, last)
            assert got[0, i, j].tolist() == want, (i, j)


@TYPES
@pytest.mark.parametrize("heads,h,d,pages,zeros", [(1, 1, 32, 40, False), (4, 2, 128, 300, False), (6, 1, 80, 70, True), (8, 4, 256, 33, True),
                                                   (3, 3, 7, 100, True),
                                                   (4, 2, 64, 1500, True)])
def test_infinite_bounds_are_the_definition(heads, h, d, pages, zeros, dtype, dev):
    """Some columns' least is -inf, some's largest is inf, some both, some the same infinity twice; queries of one sign,
    of both, and zeros, whose product with an infinity is NaN."""
    g = R.rng(pages + d)
    cache = sa.Kv4Cache.empty(pages, h, d, page_size=16, device=dev)
    bounds = torch.zeros(cache.page_bounds().shape)
    mid, half = torch.randn(pages, h, d, generator=g), torch.rand(pages, h, d, generator=g) + 1
    low, high = mid - half, mid + half
    kind = torch.randint(0, 60 * d, (pages, h, d), generator=g) // 30   # 30 of 60 d columns of each kind below 4
    low = torch.where((kind == 0) | (kind == 2), -math.inf, low)
    high = torch.where((kind == 1) | (kind == 2), math.inf, high)
    low, high = torch.where(kind == 3, math.inf, low), torch.where(kind == 3, math.inf, high)
    assert (torch.isinf(low) | torch.isinf(high)).any()
    bounds[..., 0, :d], bounds[..., 1, :d] = low, high
    bounds = bounds.to(BF16).to(dev)
    for sign in (0, 1, -1):
        q = _queries(1, 3, heads, d, dtype, 5, dev)
        q = q if sign == 0 else sign * q.abs()
        if zeros:
            q = torch.where(torch.rand(q.shape, generator=g).to(dev) < 0.1, torch.zeros_like(q), q)
        for count, first, last in ((5, 1, 1), (20, 0, 0), (pages - 1, 2, 0)):
            _check(cache, bounds, q, pages, count, first, last)


def test_bounds_of_keys_past_bfloat16(dev):
    """A column whose largest key rounds to infinity: pages stay in the order of their scores for queries that do not use
    that side, and come first for those that do."""
    pages, page, d = 20, 16, 64
    cache = sa.Kv4Cache.empty(pages, 1, d, page_size=page, device=dev)
    k = torch.randn(pages * page, 1, d, generator=R.rng(3))
    slots = torch.arange(pages * page, dtype=torch.int32, device=dev)
    cache.append(k.to(dev), k.to(dev), slots)
    # 248 * 2^120 + 15 * 1.03125 * 2^119 = 255.73 * 2^120: rounds to 256 * 2^120, bfloat16's infinity, and is below float32's
    at = 7
    cache.k_codes[at].fill_(0xFF)
    cache.k_params[at, ..., 0], cache.k_params[at, ..., 1] = 1.03125 * 2.0 ** 119, 248 * 2.0 ** 120
    bounds = cache.page_bounds()
    tables = torch.arange(pages, dtype=torch.int32, device=dev)[None]
    cache.update_page_bounds(bounds, tables, _i32([pages * page], dev), _i32([pages * page], dev))
    assert torch.isinf(bounds[at, 0, 1]).all()
    for dtype in (F32, F16, BF16):
        q = _queries(1, 1, 4, d, dtype, 1, dev)
        for x in (q, q.abs(), -q.abs()):
            _check(cache, bounds, x, pages, 4, 0, 0)
