"""Page plans and releases where something does not fit: what is taken from the free
list is in the tables, and goes back from there."""

import pytest
import torch

import serving_ref as R
import streaming_attention_b200 as sa
from streaming_attention_b200 import fast
from test_serving_path_gpu import _i32, _state

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return torch.device("cuda:0")


@pytest.fixture
def unchecked(monkeypatch):
    """Calls as they are without SA_CHECK_STATUS."""
    monkeypatch.setattr(fast, "_CHECK_STATUS", False)


def _reported(match):
    with pytest.raises(ValueError, match=match):
        sa.check_serving_status()
    sa.check_serving_status()


@pytest.mark.parametrize("requests,rows", [(1, 0), (3, 17), (40, 333), (1500, 4100)])
@pytest.mark.parametrize("per_request", [False, True])
def test_pages_of_tokens_without_rows_are_entered(requests, rows, per_request, unchecked, dev):
    """The tables and the free count are those of a plan with rows enough; the rows that
    are there hold what they hold there."""
    g = R.rng(requests)
    page, width = 16, 12
    lengths = torch.randint(0, 60, (requests,), generator=g).tolist()
    new = torch.randint(60, 130, (requests,), generator=g).tolist()
    tables, free, count = _state(lengths, page, width, requests)
    want = R.plan(lengths, new, tables, free, count, page)
    t = _i32(tables, dev)
    size = dict(per_request=7) if per_request else dict(max_tokens=rows)
    got = sa.plan_kv_pages(_i32(lengths, dev), _i32(new, dev), t, _i32(free, dev), _i32([count], dev), page_size=page, **size)
    _reported("more than the output holds")
    assert t.tolist() == want[4] and got.free_count.tolist() == [want[5]]
    assert got.lengths.tolist() == want[0] and got.offsets.tolist() == want[1]
    if per_request:
        at = [want[1][r] + i for r in range(requests) for i in range(7)]
        assert got.slots.tolist() == [want[3][i] for i in at] and got.positions.tolist() == [want[2][i] for i in at]
    else:
        assert got.slots.tolist() == want[3][:rows] and got.positions.tolist() == want[2][:rows]
    # every page is in a table or among the free ones, once
    held = [p for row in t.tolist() for p in row if p >= 0]
    assert sorted(held + free[:got.free_count.item()]) == sorted(set(held + free[:got.free_count.item()]))
    assert len(held) + got.free_count.item() == len(set(sum(([p for p in r if p >= 0] for r in tables), []))) + count


def test_page_ids_outside_the_cache_are_reported_wherever_they_stand(unchecked, dev):
    n, new, c = _i32([20], dev), _i32([1], dev), _i32([2], dev)
    plan = lambda table, free: sa.plan_kv_pages(n, new, _i32([table], dev), _i32(free, dev), c, page_size=16, max_tokens=1)  # noqa: E731
    assert plan([0, 1, -1], [2, 3]).slots.tolist() == [1 * 16 + 4]
    sa.check_serving_status(dev)
    for bad in (-7, 2, 10 ** 6):
        assert plan([0, bad, -1], [0, 1]).slots.tolist() == [-1]
        _reported("outside the cache")
    n.fill_(16)
    for bad in (-1, 2):
        p = plan([0, -1, -1], [0, bad])
        assert p.slots.tolist() == [-1] and p.tables.tolist() == [[0, -1, -1]]
        _reported("outside the cache")


def test_rows_past_31_bits_are_refused(dev):
    n = _i32([1], dev)
    with pytest.raises(ValueError, match="2\\^31"):
        sa.plan_kv_pages(n, n, n[:, None], n, n, page_size=16, max_tokens=2 ** 32)
    with pytest.raises(ValueError, match="2\\^31"):
        sa.plan_kv_pages(n, n, n[:, None], n, n, page_size=16, per_request=2 ** 31)


def test_release_empties_whole_rows(unchecked, dev):
    """Entries behind the held pages, as a plan leaves whose lengths were not taken over, do not go back to the free list."""
    n, drop = _i32([20, 20], dev), torch.tensor([True, False], device=dev)
    t = _i32([[0, 1, 5, 6], [2, 3, 7, -1]], dev)
    f, c = _i32([5, 6, 7, 8, -1, -1, -1, -1, -1], dev), _i32([4], dev)
    sa.release_kv_pages(n, t, drop, f, c, page_size=16)
    sa.check_serving_status(dev)
    assert t.tolist() == [[-1] * 4, [2, 3, 7, -1]] and n.tolist() == [0, 20]
    assert c.tolist() == [6] and f.tolist()[:6] == [5, 6, 7, 8, 0, 1]


def test_release_reports_page_ids_outside_the_cache(unchecked, dev):
    n, drop = _i32([20, 20], dev), torch.tensor([True, True], device=dev)
    t, f, c = _i32([[0, 1], [4, 99]], dev), _i32([5, 6, -1, -1, -1, -1, -1], dev), _i32([2], dev)
    sa.release_kv_pages(n, t, drop, f, c, page_size=16)
    _reported("page 99 lies outside")
    assert (t == -1).all() and n.tolist() == [0, 0] and c.tolist() == [5] and f.tolist()[:5] == [5, 6, 0, 1, 4]


def test_release_without_table_entries_empties_the_requests(unchecked, dev):
    n, e = _i32([5, 6], dev), _i32([], dev)
    sa.release_kv_pages(n, e.reshape(2, 0), torch.tensor([True, False], device=dev), e, _i32([0], dev), page_size=16)
    assert n.tolist() == [0, 6]
    sa.check_serving_status(dev)


def test_prompts_of_requests_that_hold_tokens_are_reported(unchecked, dev):
    layer = sa.StreamingWindowAttention(2, 2, 64, max_requests=3, max_length=64, window=20, page_size=16, device=dev)
    x = torch.randn(12, 2, 64, generator=R.rng(1)).to(dev)
    layer.prefill(x, x, x, _i32([5, 0, 7], dev))
    layer.prefill(x, x, x, _i32([0, 9, 0], dev))        # the others are left alone
    layer.decode(x[:3], x[:3], x[:3])
    sa.check_serving_status(dev)
    layer.prefill(x, x, x, _i32([0, 0, 4], dev))
    _reported("request 2 holds tokens already")
    layer.release(torch.tensor([False, False, True], device=dev))
    layer.prefill(x, x, x, _i32([0, 0, 4], dev))
    sa.check_serving_status(dev)
    n = _i32([1], dev)
    with pytest.raises(ValueError, match="packed"):
        sa.plan_kv_pages(n, n, n[:, None], n, n, page_size=16, per_request=1, prompts=True)
