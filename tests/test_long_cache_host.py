"""Refusals of the entry points for long caches, on the CPU: no launch is made."""

import ctypes

import pytest
import torch

import streaming_attention_b200 as sa
from streaming_attention_b200 import _lib, _serving, kv4
from test_kv4_host import _tensors


@pytest.fixture(autouse=True)
def no_launch(monkeypatch):
    monkeypatch.setattr(_serving, "device_of", lambda first, *others: first.device)
    monkeypatch.setattr(_serving, "launch", lambda *a: pytest.fail("launched"))
    assert kv4.S is _serving


@pytest.fixture
def cache():
    return sa.Kv4Cache(*_tensors(4), 64)


def _i(*shape):
    return torch.zeros(shape, dtype=torch.int32)


Q = torch.zeros(3, 4, 64)


def test_attend_refuses_weights_that_do_not_fit(cache):
    good = cache.token_weights()
    assert good.shape == (4, 2, 16) and good.dtype == torch.float32
    for bad in (good.double(), good[:3], good[..., :15], torch.stack([good, good], -1)[..., 0], good.expand(4, 2, 16)[:, :, ::1].transpose(0, 1)):
        with pytest.raises(ValueError, match="weights must be"):
            cache.attend(Q, _i(3, 2), _i(3), weights=bad)
        with pytest.raises(ValueError, match="weights must be"):
            cache.reset_weights(bad, _i(1))
        with pytest.raises(ValueError, match="weights must be"):
            cache.evict(bad, _i(3), _i(3, 2), _i(4), _i(1), keep=3)
    with pytest.raises(ValueError, match=r"slots must be \[T\]"):
        cache.reset_weights(good, _i(1, 1))
    with pytest.raises(ValueError, match="slots must be int32"):
        cache.reset_weights(good, torch.zeros(1))


def test_attend_shared_refuses(cache):
    with pytest.raises(ValueError, match=r"prefix_table must be \[W0\]"):
        cache.attend_shared(Q, _i(1, 2), _i(1), _i(3, 2), _i(3))
    with pytest.raises(ValueError, match="prefix_table must be int32"):
        cache.attend_shared(Q, _i(2).long(), _i(1), _i(3, 2), _i(3))
    with pytest.raises(ValueError, match="prefix_length must have shape"):
        cache.attend_shared(Q, _i(2), _i(2), _i(3, 2), _i(3))
    with pytest.raises(ValueError, match="head width 64"):
        cache.attend_shared(Q[..., :32], _i(2), _i(1), _i(3, 2), _i(3))
    with pytest.raises(ValueError, match="multiple of 2 heads"):
        cache.attend_shared(Q[:, :3], _i(2), _i(1), _i(3, 2), _i(3))
    with pytest.raises(ValueError, match="tables must be"):
        cache.attend_shared(Q, _i(2), _i(1), _i(4, 2), _i(4))
    with pytest.raises(ValueError, match="window must be positive"):
        cache.attend_shared(Q, _i(2), _i(1), _i(3, 2), _i(3), window=0)
    with pytest.raises(ValueError, match="unsupported dtype"):
        cache.attend_shared(Q.double(), _i(2), _i(1), _i(3, 2), _i(3))


def test_attend_pages_refuses(cache):
    for bad in (_i(3, 2), _i(3, 1, 2, 5), _i(3, 3, 5), _i(2, 2, 5)):
        with pytest.raises(ValueError, match="pages must"):
            cache.attend_pages(Q, _i(3, 2), _i(3), bad)
    with pytest.raises(ValueError, match="pages must"):
        cache.attend_pages(Q[:, None], _i(3, 2), _i(3), _i(3, 2, 5))
    with pytest.raises(ValueError, match="pages must be int32"):
        cache.attend_pages(Q, _i(3, 2), _i(3), _i(3, 2, 5).long())


def test_bounds_and_selection_refuse(cache):
    good = cache.page_bounds()
    assert good.shape == (4, 2, 2, 64) and good.dtype == torch.bfloat16
    for bad in (good.float(), good[:3], good[..., :32], torch.stack([good, good], -1)[..., 0]):
        with pytest.raises(ValueError, match="bounds must be"):
            cache.update_page_bounds(bad, _i(3, 2), _i(3), _i(3))
        with pytest.raises(ValueError, match="bounds must be"):
            cache.select_pages(Q, bad, _i(3, 2), _i(3), count=2)
    with pytest.raises(ValueError, match="new must have shape"):
        cache.update_page_bounds(good, _i(3, 2), _i(3), _i(2))
    for kw, match in ((dict(count=1), "no more than count"), (dict(count=4, first=-1), "non-negative"),
                      (dict(count=4, last=-1), "non-negative"), (dict(count=-1, first=0, last=0), "count must lie"),
                      (dict(count=2.5), "whole number"), (dict(count=4, first=3, last=2), "no more than count")):
        with pytest.raises(ValueError, match=match):
            cache.select_pages(Q, good, _i(3, 2), _i(3), **kw)


def test_evict_refuses(cache):
    w = cache.token_weights()

    def call(lengths=_i(3), tables=_i(3, 2), free=_i(4), count=_i(1), **kw):
        cache.evict(w, lengths, tables, free, count, **kw)

    for kw, match in ((dict(keep=0), "keep must be positive"), (dict(keep=4, limit=3), "limit no less"),
                      (dict(keep=4, first=3, last=2), "no more than keep"), (dict(keep=4, first=-1), "non-negative"),
                      (dict(keep=4, last=-1), "non-negative"), (dict(keep=1.5), "whole number"),
                      (dict(keep=4, limit=2 ** 31), "limit no less"),
                      (dict(keep=4, lengths=_i(2)), "lengths must have shape"), (dict(keep=4, tables=_i(3)), r"tables must be \[R,W\]"),
                      (dict(keep=4, free=_i(1, 4)), r"free_pages must be \[F\]"), (dict(keep=4, count=_i(2)), "free_count must have"),
                      (dict(keep=4, tables=_i(2, 3).T), "contiguous"), (dict(keep=4, lengths=_i(6)[::2]), "contiguous")):
        with pytest.raises(ValueError, match=match):
            call(**kw)


def test_calls_without_rows_launch_nothing(cache):
    w, b = cache.token_weights(), cache.page_bounds()
    assert cache.attend(Q[:0], _i(0, 2), _i(0), weights=w).shape == (0, 4, 64)
    assert cache.attend_shared(Q[:0], _i(2), _i(1), _i(0, 2), _i(0)).shape == (0, 4, 64)
    assert cache.attend_pages(Q[:0], _i(0, 2), _i(0), _i(0, 2, 5)).shape == (0, 4, 64)
    assert cache.select_pages(Q[:0], b, _i(0, 2), _i(0), count=3).shape == (0, 2, 3)
    assert cache.select_pages(Q, b, _i(3, 2), _i(3), count=0, first=0, last=0).shape == (3, 2, 0)
    cache.update_page_bounds(b, _i(0, 2), _i(0), _i(0))
    cache.reset_weights(w, _i(0))
    kept, dropped = cache.evict(w, _i(0), _i(0, 2), _i(4), _i(1), keep=3)
    assert kept.shape == (0, 2, 3) and dropped.shape == (0,)


def test_sizes_are_refused_by_the_library():
    lib, size = _lib.load(), ctypes.c_size_t(0)
    shared = lambda *a: lib.sa_kv4_attend_shared_workspace_size(*a, 0, 0, 0, ctypes.byref(size))  # noqa: E731
    assert shared(2, 16, 64, 3, 1, 4, 10) == 0 and size.value > 0
    assert shared(2, 16, 64, 3, 1, 5, 10) == _lib.SA_ERR_INVALID_ARG
    assert shared(2, 17, 64, 3, 1, 4, 10) == _lib.SA_ERR_INVALID_ARG
    assert shared(2, 16, 300, 3, 1, 4, 10) == _lib.SA_ERR_INVALID_ARG
    assert shared(2, 16, 64, 65535, 1, 8, 10) == _lib.SA_ERR_UNSUPPORTED
    assert shared(2, 16, 64, 3, 1, 4, 1 << 28) == _lib.SA_ERR_UNSUPPORTED
    weigh = lambda *a: lib.sa_kv4_attend_weigh_workspace_size(*a, ctypes.byref(size))  # noqa: E731
    assert weigh(2, 16, 3, 1, 4, 10, 0, 0) == 0 and size.value > 0
    whole = size.value
    assert weigh(2, 16, 3, 1, 4, 10, 20, 3) == 0 and size.value < whole
    assert weigh(2, 16, 3, 1, 4, 10, -1, 0) == _lib.SA_ERR_INVALID_ARG
