"""Sizes that the entry points for long caches refuse, and that a refused call leaves everything as it was."""

import ctypes

import pytest
import torch

import streaming_attention_b200 as sa
from streaming_attention_b200 import _lib
from test_kv4_gpu import _filled
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
