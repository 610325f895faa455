"""What a Kv4Cache hands to the kernels, on the CPU: the launches are caught before
they reach the library."""

import pytest
import torch

import streaming_attention_b200 as sa
from streaming_attention_b200 import kv4


@pytest.fixture
def calls(monkeypatch):
    got = []
    monkeypatch.setattr(kv4.S, "device_of", lambda first, *others: first.device)
    monkeypatch.setattr(kv4.S, "launch", lambda dev, name, *args: got.append((name, args)))
    return got


def _tensors(pages, heads=2, page=16, half=32):
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    b16 = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    return (u8(pages, heads, page, half), b16(pages, heads, page, 2), u8(pages, heads, page // 4, half, 4),
            b16(pages, heads, page, 2))


def _use(cache):
    x, i = torch.zeros(1, 2, 64), torch.zeros(1, dtype=torch.int32)
    cache.append(x, x, i)
    cache.read(i)
    cache.attend(x, i[:, None], i)


NAMES = ("k_codes", "k_params", "v_codes", "v_params")


def test_replaced_tensors_are_the_ones_used(calls):
    cache = sa.Kv4Cache(*_tensors(4), 64)
    _use(cache)
    new = _tensors(9)
    for name, t in zip(NAMES, new):
        setattr(cache, name, t)
    _use(cache)
    assert [n for n, _ in calls] == ["sa_kv4_append", "sa_kv4_read", "sa_kv4_attend"] * 2
    for _, args in calls[3:]:
        assert args[:8] == (*(t.data_ptr() for t in new), 9, 2, 16, 64)
    assert cache.num_pages == 9


def test_replaced_memory_is_the_one_used(calls):
    cache = sa.Kv4Cache(*_tensors(4), 64)
    for name in NAMES:
        t = getattr(cache, name)
        t.data = t.data.clone()
    _use(cache)
    for _, args in calls:
        assert args[:4] == tuple(getattr(cache, n).data_ptr() for n in NAMES)


@pytest.mark.parametrize("name", NAMES)
def test_tensors_that_do_not_fit_are_refused_at_the_next_call(name, calls):
    x, i = torch.zeros(1, 2, 64), torch.zeros(1, dtype=torch.int32)
    for make in (lambda t: torch.cat([t, t]), lambda t: t.float(), lambda t: torch.stack([t, t], -1)[..., 0]):
        cache = sa.Kv4Cache(*_tensors(4), 64)
        setattr(cache, name, make(getattr(cache, name)))
        for call in (lambda: cache.append(x, x, i), lambda: cache.read(i), lambda: cache.attend(x, i[:, None], i)):
            with pytest.raises(ValueError, match="must be"):
                call()
    assert not calls
