"""Sizes that the entry points for long caches refuse, and that a refused call leaves everything as it was."""

import ctypes

import pytest
import torch

import streaming_attention_b200 as sa
from streaming_attention_b200 import _lib, _serving
from test_kv4_gpu import _filled
from test_kv4_host import _tensors
from test_long_cache_gpu import F32


def _evict(requests, width=1, keep=1, limit=1, page_size=16, at=0x10000):
    """The C entry point with addresses that are never reached: what is tested is refused before a launch."""
    p = ctypes.c_void_p(at)
    return _lib.load().sa_kv4_evict(p, p, p, p, 4, 1, page_size, 64, p, p, p, p, p, requests, width, 1, keep, limit, 0, 0, p, p, None)


def test_evict_refuses_many_requests_before_it_moves_anything():
    for requests in (16385, 65535):
        assert _evict(requests) == _lib.SA_ERR_UNSUPPORTED
        assert "16384 requests" in _lib.load().sa_last_error().decode()
    assert _evict(65536) == _lib.SA_ERR_UNSUPPORTED


def test_sizes_near_31_bits_are_refused():
    assert _evict(1, width=(1 << 26) + 1) == _lib.SA_ERR_UNSUPPORTED and "2^30 tokens" in _lib.load().sa_last_error().decode()
    assert _evict(1, keep=(1 << 30) + 1, limit=2 ** 31 - 1) == _lib.SA_ERR_UNSUPPORTED
    lib, p = _lib.load(), ctypes.c_void_p(0x10000)
    strides = (ctypes.c_int64 * 3)(64, 64, 64)
    for count in ((1 << 30) + 1, 2 ** 31 - 1):
        assert lib.sa_kv4_select_pages(p, 4, 1, 16, 64, p, strides, p, p, 1, 1, 1, 1, count, 0, 0, 0, p, None) == _lib.SA_ERR_UNSUPPORTED
        assert lib.sa_kv4_attend_pages(p, p, p, p, 4, 1, 16, 64, p, p, strides, p, p, p, count, 1, 1, 1, 1, 1.0, 0, None) == _lib.SA_ERR_UNSUPPORTED
        assert "2^30" in lib.sa_last_error().decode()


def test_sizes_past_31_bits_do_not_reach_the_library(monkeypatch):
    """Expanded tensors of a size that a 32-bit argument would cut off to 3."""
    monkeypatch.setattr(_serving, "device_of", lambda first, *others: first.device)
    monkeypatch.setattr(_serving, "launch", lambda *a: pytest.fail("launched"))
    far = 2 ** 32 + 3
    cache = sa.Kv4Cache(*_tensors(4), 64)
    i = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    q, wide = torch.zeros(1, 2, 64), i(1, 1).expand(1, far)
    weights, bounds = cache.token_weights(), cache.page_bounds()
    for call in (lambda: cache.attend(q, wide, i(1)), lambda: cache.attend(q, wide, i(1), weights=weights),
                 lambda: cache.attend_shared(q, wide[0], i(1), i(1, 1), i(1)), lambda: cache.attend_shared(q, i(1), i(1), wide, i(1)),
                 lambda: cache.attend_pages(q, i(1, 1), i(1), i(1, 2, 1).expand(1, 2, far)),
                 lambda: cache.attend_pages(q, wide, i(1), i(1, 2, 1)),
                 lambda: cache.update_page_bounds(bounds, wide, i(1), i(1)),
                 lambda: cache.select_pages(q, bounds, wide, i(1), count=2),
                 lambda: cache.evict(weights, i(1), wide, i(1), i(1), keep=1),
                 lambda: cache.evict(weights, i(1), i(1, 1), i(1).expand(far), i(1), keep=1)):
        with pytest.raises(ValueError, match=r"below 2\^31"):
            call()
    with pytest.raises(ValueError, match="count must lie"):
        cache.select_pages(q, bounds, i(1, 1), i(1), count=(1 << 30) + 1)


@pytest.mark.gpu
def test_a_refused_eviction_changes_nothing():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    dev, requests = torch.device("cuda:0"), 16385
    cache, tables, lens, _, _ = _filled(dev, [100], 1, 64, 16, F32, 1)
    weights = torch.rand(cache.token_weights().shape, device=dev)
    lengths = torch.zeros(requests, dtype=torch.int32, device=dev)
    lengths[:1] = lens
    wide = torch.full((requests, tables.shape[1]), -1, dtype=torch.int32, device=dev)
    wide[:1] = tables
    free, count = torch.zeros(99, dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    state = (cache.k_codes, cache.k_params, cache.v_codes, cache.v_params, weights, lengths, wide, free, count)
    bits = lambda t: t.view(torch.int16) if t.dtype == torch.bfloat16 else t  # noqa: E731  (NaN in slots of nobody)
    before = [bits(t).clone() for t in state]
    with pytest.raises(NotImplementedError, match="16384 requests"):
        cache.evict(weights, lengths, wide, free, count, keep=10)
    assert all(torch.equal(bits(s), t) for s, t in zip(state, before))
    # and the most that one call takes
    kept, dropped = cache.evict(weights, lengths[:-1], wide[:-1], free, count, keep=10)
    assert lengths[:2].tolist() == [10, 0] and dropped.tolist() == [90] + [0] * 16383 and count.item() == 6
    assert (kept[1:] == -1).all()
