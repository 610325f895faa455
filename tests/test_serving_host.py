"""Refusals of the serving entry points that need no GPU: the C ABI's argument
checks return before any CUDA call."""

import ctypes

import pytest

import streaming_attention_b200 as sa
from streaming_attention_b200 import _lib

INV, UNS = _lib.SA_ERR_INVALID_ARG, _lib.SA_ERR_UNSUPPORTED
P = 1 << 20   # stands for a pointer; never followed


def _strides(n):
    return (ctypes.c_int64 * n)(*([64] * n))


def _window(**kw):
    a = dict(q=P, k=P, v=P, out=P, strides=_strides(12), batch=1, heads=4, kv_heads=2, n=8, m=8, d=64, dv=64, window=4, sinks=0,
             scale=1.0, dtype=2, cu_q=None, cu_k=None, zero=0, ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    return _lib.load().sa_window_attention(*a.values())


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=3), INV), (dict(heads=3), INV), (dict(kv_heads=0), INV), (dict(heads=0), INV), (dict(n=9), INV), (dict(n=-1), INV),
    (dict(d=0), INV), (dict(d=257), INV), (dict(dv=257), INV), (dict(window=-1), INV), (dict(sinks=-1), INV), (dict(cu_q=P), INV),
    (dict(m=1 << 31, n=1), UNS), (dict(q=None), INV), (dict(out=None), INV), (dict(strides=None), INV), (dict(v=None), INV),
    (dict(n=0), _lib.SA_OK), (dict(batch=0), _lib.SA_OK)])
def test_window_arguments(kw, rc):
    assert _window(**kw) == rc


def _cache(**kw):
    a = dict(kc=P, kp=P, vc=P, vp=P, pages=4, heads=2, page=16, d=64)
    a.update(kw)
    return a


CACHE_BAD = [(dict(page=24), INV), (dict(page=8), INV), (dict(page=512), INV), (dict(pages=0), INV), (dict(heads=0), INV),
             (dict(d=0), INV), (dict(d=300), INV), (dict(kc=None), INV), (dict(vp=None), INV), (dict(kc=P + 8), INV),
             (dict(pages=1 << 27), UNS)]


@pytest.mark.parametrize("kw,rc", CACHE_BAD)
def test_cache_arguments(kw, rc):
    lib, c = _lib.load(), _cache(**kw)
    assert lib.sa_kv4_append(*c.values(), P, P, _strides(4), P, 3, 0, None) == rc
    assert lib.sa_kv4_read(*c.values(), P, P, P, 3, 0, None) == rc
    assert lib.sa_kv4_attend(*c.values(), P, P, _strides(3), P, P, 1, 1, 4, 2, 0, 0, 1.0, 0, None) == rc


def test_cache_call_arguments():
    lib, c = _lib.load(), _cache()
    append = lambda *a: lib.sa_kv4_append(*c.values(), *a)  # noqa: E731
    assert append(P, P, _strides(4), P, 3, 7, None) == INV
    assert append(P, P, _strides(4), P, -1, 0, None) == INV
    assert append(P, None, _strides(4), P, 1, 0, None) == INV
    assert append(P, P, None, P, 1, 0, None) == INV
    assert append(None, None, None, None, 0, 0, None) == _lib.SA_OK
    attend = lambda q=P, out=P, st=_strides(3), t=P, l=P, r=1, n=1, h=4, w=2, win=0, s=0, dt=0: lib.sa_kv4_attend(  # noqa: E731
        *c.values(), q, out, st, t, l, r, n, h, w, win, s, 1.0, dt, None)
    for kw, rc in ((dict(h=3), INV), (dict(r=-1), INV), (dict(n=-1), INV), (dict(w=-1), INV), (dict(win=-1), INV), (dict(s=-1), INV),
                   (dict(dt=9), INV), (dict(q=None), INV), (dict(t=None), INV), (dict(l=None), INV), (dict(st=None), INV),
                   (dict(r=65536), UNS), (dict(n=20000), UNS), (dict(r=0), _lib.SA_OK), (dict(n=0), _lib.SA_OK)):
        assert attend(**kw) == rc, kw


def test_plan_arguments():
    plan = lambda requests=2, width=4, free=8, page=16, cap=5, per=0, lengths=P, tables=P, slots=P: _lib.load().sa_plan_kv_pages(  # noqa: E731
        lengths, P, tables, P, P, requests, width, free, page, cap, per, P, P, P, slots, P, None)
    for kw, rc in ((dict(page=17), INV), (dict(requests=-1), INV), (dict(width=-1), INV), (dict(free=-1), INV), (dict(cap=-1), INV),
                   (dict(per=-1), INV), (dict(per=3), INV), (dict(lengths=None), INV), (dict(tables=None), INV), (dict(slots=None), INV),
                   (dict(requests=1 << 20, width=1 << 12), UNS), (dict(free=1 << 28), UNS), (dict(requests=16385), UNS)):
        assert plan(**kw) == rc, kw


def test_rotary_arguments():
    call = lambda q=P, pos=P, f=P, st=_strides(8), t=2, h=4, hk=2, d=64, half=32, dt=0: _lib.load().sa_qk_norm_rotary(  # noqa: E731
        q, P, P, P, pos, None, None, f, st, t, h, hk, d, half, 1e-6, 0, 0, dt, None)
    for kw, rc in ((dict(dt=5), INV), (dict(t=-1), INV), (dict(h=0, hk=0), INV), (dict(h=-1), INV), (dict(d=0), INV), (dict(d=257), INV),
                   (dict(half=33), INV), (dict(half=-1), INV), (dict(q=None), INV), (dict(pos=None), INV), (dict(f=None), INV),
                   (dict(st=None), INV), (dict(t=0), _lib.SA_OK)):
        assert call(**kw) == rc, kw


def test_cpu_tensors_and_missing_devices_are_refused():
    import torch
    x = torch.zeros(1, 2, 4, 64)
    with pytest.raises(ValueError, match="CUDA tensors"):
        sa.sliding_window_attention(x, x, x, window=2)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensors"):
        sa.plan_kv_pages(i, i, i[:, None], i, i, page_size=16, max_tokens=1)
    with pytest.raises(ValueError, match="CUDA tensors"):
        sa.qk_norm_rotary(x[0], x[0], i, None, None, sa.rotary_frequencies(64))
    if not torch.cuda.is_available():
        with pytest.raises(ValueError, match="need a CUDA device"):
            sa.Kv4Cache.empty(2, 2, 64)


def test_rotary_frequencies():
    f = sa.rotary_frequencies(8, base=100.0)
    assert f.tolist() == pytest.approx([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], rel=1e-15)
    assert sa.rotary_frequencies(0).numel() == 0


def test_windows_and_first_tokens_are_whole_numbers():
    from streaming_attention_b200 import _serving as S
    nan, inf = float("nan"), float("inf")
    for window, sinks, match in ((0.5, 0, "window must be a whole"), (1.5, 0, "window must be a whole"), (nan, 0, "window must be a whole"),
                                 (inf, 0, "window must be a whole"), ("4", 0, "window must be a whole"), (4, 0.5, "sinks must be a whole"),
                                 (4, None, "sinks must be a whole"), (0, 0, "window must be positive"), (-1.0, 0, "window must be positive"),
                                 (4, -1, "sinks must be non-negative")):
        with pytest.raises(ValueError, match=match):
            S.check_window(window, sinks)
        with pytest.raises(ValueError, match=match):
            sa.StreamingWindowAttention(2, 2, 64, max_requests=1, max_length=10, window=window, sinks=sinks)
    assert S.check_window(None, 3) == (0, 3) and S.check_window(7.0, 0) == (7, 0) and S.check_window(2 ** 64, 2 ** 50) == (1 << 40, 1 << 40)


def test_prompt_plan_arguments():
    plan = lambda requests=2, width=4, free=8, page=16, cap=5, lengths=P, tables=P, slots=P: _lib.load().sa_plan_kv_prompts(  # noqa: E731
        lengths, P, tables, P, P, requests, width, free, page, cap, P, P, P, slots, P, None)
    for kw, rc in ((dict(page=17), INV), (dict(requests=-1), INV), (dict(width=-1), INV), (dict(free=-1), INV), (dict(cap=-1), INV),
                   (dict(lengths=None), INV), (dict(tables=None), INV), (dict(slots=None), INV), (dict(requests=1 << 20, width=1 << 12), UNS),
                   (dict(free=1 << 28), UNS), (dict(requests=16385), UNS)):
        assert plan(**kw) == rc, kw
