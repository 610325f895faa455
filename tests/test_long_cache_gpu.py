"""Long caches: attention behind a shared prefix and over selected pages, bounds and
selection, accumulated weights and eviction, against their float64 definitions.
Attention errors are held to serving_ref.attention_bound; what is chosen, moved or
counted is equal."""

import math

import pytest
import torch

import long_cache_ref as L
import serving_ref as R
import streaming_attention_b200 as sa
from test_kv4_gpu import _filled

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
# rounding of the probabilities: 16 bits kept; over a shared prefix those of 16-bit queries and the
# values are rounded to float16: half a step (2^-11) of each term p v from either, 2^-10 in all
P_HALF = {F32: 0.0, F16: 2.0 ** -16, BF16: 2.0 ** -16}
P_SHARED = {F32: 0.0, F16: 2.0 ** -10, BF16: 2.0 ** -10}


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return torch.device("cuda:0")


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _queries(r, n, heads, d, dtype, seed, dev):
    return (torch.randn(r, n, heads, d, generator=R.rng(seed)) * 1.5).to(dtype).to(dev)


def _close(out, ref, spread, score, d, keys, p_half, span=None):
    dtype = out.dtype
    span = R.code_span(dtype) if span is None else span
    R.assert_close(out, ref, R.attention_bound(ref, spread, span * score, d, max(keys, 1), dtype, p_half))


def _one_step(a, b):
    """Results of bfloat16 whose sums were added in another order: float32 sums that differ by less than 2^-14 (2^-16 of
    values below 4), each rounded, are a step apart at most (2^-7 of the value: twice half a step)."""
    a, b = a.double(), b.double()
    assert ((a - b).abs() <= 2 * R.HALF[BF16] * torch.maximum(a.abs(), b.abs()) + 2.0 ** -14).all()


# ------------------------------------------------------------- shared prefix

SHARED = [
    # prefix, own lengths, heads, kv heads, n, d, page, window, sinks
    (1, [1], 1, 1, 1, 64, 16, None, 0),
    (17, [5, 0, 1, 40], 4, 2, 1, 128, 16, None, 0),
    (300, [3, 2, 1, 0, 9], 6, 2, 3, 64, 32, None, 0),
    (1000, [64, 65, 200], 8, 1, 1, 128, 64, 150, 4),
    (1000, [64, 65, 1200], 8, 2, 2, 80, 64, 1100, 700),
    (257, [33] * 40, 8, 1, 1, 128, 128, None, 0),
    (1537, [20] * 17 + [0] + [31] * 16, 16, 2, 2, 64, 16, None, 0),
    (2049, [7, 70, 300] * 30, 4, 4, 1, 128, 64, 1000, 130),
    (700, [90, 15], 5, 1, 1, 127, 256, 1, 1),
    (515, [10, 20, 30], 24, 1, 2, 256, 16, 200, 530),
    (90, [11, 12], 2, 2, 1, 7, 16, 20, 3),
    (6000, [500, 1], 12, 4, 4, 96, 64, None, 0),
    (0, [40, 3], 4, 2, 1, 64, 16, None, 0),
    (5000, [13] * 70, 8, 2, 1, 32, 64, 3000, 2),
    (9001, [3] * 40, 64, 8, 1, 64, 64, None, 0),    # long chains of tiles in one part
    (4100, [5, 6] * 33, 96, 8, 2, 32, 32, None, 0),
    (900, [5] * 40, 8, 1, 1, 64, 256, None, 0),
    (700, [9] * 40, 5, 1, 1, 127, 64, 300, 33),
    (200, [9, 30] * 9, 10, 2, 1, 50, 16, 60, 3),
]


@TYPES
@pytest.mark.parametrize("case", range(len(SHARED)))
def test_shared_prefix_matches_definition(case, dtype, dev):
    prefix, lengths, heads, h, n, d, page, window, sinks = SHARED[case]
    cache, tables, lens, ks, vs = _filled(dev, [prefix] + lengths, h, d, page, F32, case)
    q = _queries(len(lengths), n, heads, d, dtype, case + 70, dev)
    out = cache.attend_shared(q, tables[0], lens[:1], tables[1:], lens[1:], window=window, sinks=sinks)
    assert out.shape == q.shape and out.dtype == dtype
    for r, x in enumerate(lengths):
        k, v = torch.cat([ks[0], ks[r + 1]]), torch.cat([vs[0], vs[r + 1]])
        sees = R.visible(n, prefix + x, window, sinks)
        sees[:max(0, n - x)] = False   # only a request's own tokens ask
        ref, spread, score, _ = L.attend(q[r].cpu().double(), k, v, sees, 1 / math.sqrt(d))
        _close(out[r], ref, spread, score, d, prefix + x, P_SHARED[dtype])
    if n == 1:
        one = cache.attend_shared(q[:, 0], tables[0], lens[:1], tables[1:], lens[1:], window=window, sinks=sinks)
        assert torch.equal(one, out[:, 0])
    # the same bits every time
    assert torch.equal(out, cache.attend_shared(q, tables[0], lens[:1], tables[1:], lens[1:], window=window, sinks=sinks))


@pytest.mark.parametrize("prefix", [1, 15, 16, 31, 63, 64, 65, 127, 128, 129, 255, 256, 257, 383, 385])
def test_shared_prefix_lengths(prefix, dev):
    lengths = [9] * 40
    cache, tables, lens, ks, vs = _filled(dev, [prefix] + lengths, 1, 128, 64, F32, prefix)
    q = _queries(40, 1, 4, 128, BF16, prefix, dev)
    out = cache.attend_shared(q, tables[0], lens[:1], tables[1:], lens[1:])
    for r, x in enumerate(lengths):
        ref, spread, score, _ = L.attend(q[r].cpu().double(), torch.cat([ks[0], ks[r + 1]]), torch.cat([vs[0], vs[r + 1]]),
                                         R.visible(1, prefix + x, None, 0), 1 / math.sqrt(128))
        _close(out[r], ref, spread, score, 128, prefix + x, P_SHARED[BF16])


@TYPES
def test_shared_prefix_strides_and_scale(dtype, dev):
    """Queries as a slice of a projection; a scale that is negative, or zero."""
    cache, tables, lens, ks, vs = _filled(dev, [200, 30, 40, 50], 2, 64, 16, F32, 5)
    wide = _queries(3, 2, 12, 64, dtype, 6, dev)
    q = wide[:, :, 4:8]
    for scale in (0.3, -0.1, 0.0):
        out = cache.attend_shared(q, tables[0], lens[:1], tables[1:], lens[1:], scale=scale)
        assert torch.equal(out, cache.attend_shared(q.contiguous(), tables[0], lens[:1], tables[1:], lens[1:], scale=scale))
        for r, x in enumerate([30, 40, 50]):
            ref, spread, score, _ = L.attend(q[r].cpu().double(), torch.cat([ks[0], ks[r + 1]]),
                                             torch.cat([vs[0], vs[r + 1]]), R.visible(2, 200 + x, None, 0), scale)
            _close(out[r], ref, spread, score, 64, 200 + x, P_SHARED[dtype])


@TYPES
@pytest.mark.parametrize("requests", [3, 70])
def test_shared_prefix_scores_far_apart_and_flat(requests, dtype, dev):
    """Scores of several hundred, whose maximum moves from tile to tile, and equal ones; constant rows (scale 0)."""
    g, n_prefix, d = R.rng(8), 900, 64
    for size in (0.0, 1.0, 60.0):
        cache = sa.Kv4Cache.empty(20 + requests, 1, d, page_size=64, device=dev)
        k = torch.randn(n_prefix + requests, 1, d, generator=g) * size
        v = torch.randn(n_prefix + requests, 1, d, generator=g) + 2
        k[7], v[300] = 1.25, -0.75   # rows without a span
        slots = torch.arange(n_prefix + requests, dtype=torch.int32)
        slots[n_prefix:] = (15 + torch.arange(requests, dtype=torch.int32)) * 64
        cache.append(k.to(dev), v.to(dev), slots.to(dev))
        rk, rv = (x.cpu().double() for x in cache.read(slots.to(dev)))
        q = _queries(requests, 1, 2, d, dtype, 3, dev)
        out = cache.attend_shared(q, _i32(list(range(15)), dev), _i32([n_prefix], dev), _i32([[15 + r] for r in range(requests)], dev),
                                  _i32([1] * requests, dev))
        for r in range(0, requests, 7):
            at = list(range(n_prefix)) + [n_prefix + r]
            ref, spread, score, _ = L.attend(q[r].cpu().double(), rk[at], rv[at], R.visible(1, n_prefix + 1, None, 0), 0.125)
            _close(out[r], ref, spread, score, d, n_prefix + 1, P_SHARED[dtype])


@pytest.mark.parametrize("requests", [2, 70])
def test_shared_prefix_bad_pages_and_nan(requests, dev):
    """NaN rows reach who sees them and nobody else; a page id outside the cache is reported and hidden."""
    lengths = [20] * requests
    cache, tables, lens, ks, vs = _filled(dev, [300] + lengths, 1, 64, 16, F32, 2)
    q = _queries(requests, 1, 2, 64, BF16, 1, dev)
    clean = cache.attend_shared(q, tables[0], lens[:1], tables[1:], lens[1:], window=100, sinks=2)
    page = tables[0, 5].item()   # tokens 80..95: hidden by the window
    cache.k_params[page] = float("nan")
    cache.v_params[page] = float("nan")
    assert torch.equal(clean, cache.attend_shared(q, tables[0], lens[:1], tables[1:], lens[1:], window=100, sinks=2))
    assert torch.isnan(cache.attend_shared(q, tables[0], lens[:1], tables[1:], lens[1:])).all()
    table = tables[0].clone()
    table[5] = 10 ** 6
    with pytest.raises(ValueError, match="outside the cache"):
        cache.attend_shared(q, table, lens[:1], tables[1:], lens[1:])
    with pytest.raises(ValueError, match="longer than its table"):
        cache.attend_shared(q, tables[0, :3], lens[:1], tables[1:], lens[1:])


def _shared_case(dev, requests, k, v, window, sinks, dtype, q_scale=1.0, own=5, seed=1):
    """Prefix rows k, v [P,1,64] and `own` tokens of each request, of the same size; checks every request."""
    prefix, g = k.shape[0], R.rng(seed)
    pages = -(-prefix // 64)
    cache = sa.Kv4Cache.empty(pages + requests, 1, 64, page_size=64, device=dev)
    own_k, own_v = (torch.randn(requests * own, 1, 64, generator=g) * x[:3].abs().median() for x in (k, v))
    slots = torch.cat([torch.arange(prefix), ((pages + torch.arange(requests))[:, None] * 64 + torch.arange(own)).flatten()]).to(torch.int32)
    cache.append(torch.cat([k, own_k]).to(dev), torch.cat([v, own_v]).to(dev), slots.to(dev))
    rk, rv = (x.cpu().double() for x in cache.read(slots.to(dev)))
    q = (_queries(requests, 1, 2, 64, F32, seed + 1, dev) * q_scale).to(dtype)
    out = cache.attend_shared(q, torch.arange(pages, dtype=torch.int32, device=dev), _i32([prefix], dev),
                              (pages + torch.arange(requests, dtype=torch.int32, device=dev))[:, None], _i32([own] * requests, dev),
                              window=window, sinks=sinks)
    for r in range(requests):
        at = list(range(prefix)) + list(range(prefix + r * own, prefix + (r + 1) * own))
        ref, spread, score, _ = L.attend(q[r].cpu().double(), torch.nan_to_num(rk[at]), torch.nan_to_num(rv[at]),
                                         R.visible(1, prefix + own, window, sinks), 0.125)
        _close(out[r], ref, spread, score, 64, prefix + own, P_SHARED[dtype])


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("k_size,v_size,q_size", [(1e-15, 1e20, 1.0), (1e15, 1e-20, 1e-4), (1e-30, 1e-30, 1.0), (1.0, 1.0, 1e-5)])
def test_shared_prefix_of_any_size(k_size, v_size, q_size, dtype, dev):
    if dtype == F16 and v_size > 1:
        v_size = 1e3   # float16 results
    g = R.rng(4)
    _shared_case(dev, 40, torch.randn(500, 1, 64, generator=g) * k_size, torch.randn(500, 1, 64, generator=g) * v_size, None, 0,
                 dtype, q_size)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("which", ["k", "v"])
def test_shared_prefix_of_sizes_far_apart(which, dtype, dev):
    """One token's row a million times the others, and one a millionth of them: seen, with little weight."""
    g = R.rng(4)
    k, v = torch.randn(500, 1, 64, generator=g), torch.randn(500, 1, 64, generator=g)
    if which == "k":
        k[100] *= 1e-3   # scores that say nothing, beside those of the others
        k[200] *= 1e-7
    else:
        v[100] *= 1e4
        v[200] *= 1e-6
    _shared_case(dev, 40, k, v, None, 0, dtype)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("value", [1e30, 3e38, float("inf"), float("nan")])
def test_shared_prefix_hidden_rows_of_any_size(value, dtype, dev):
    """What no query sees, in a tile whose other tokens are seen, changes nothing."""
    g = R.rng(4)
    k, v = torch.randn(500, 1, 64, generator=g), torch.randn(500, 1, 64, generator=g)
    k[3:390], v[3:390] = value, value   # 505 - 110 = 395: visible from there on, and tokens 0..2
    _shared_case(dev, 40, k, v, 110, 3, dtype)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_shared_prefix_rows_that_only_some_see(dtype, dev):
    """Requests of other lengths: the shorter see a token of 1e25 or NaN, the longer ones' windows end behind it."""
    g, requests, prefix, d = R.rng(9), 40, 700, 64
    for bad in (1e25, float("nan")):
        lengths = [3 + 2 * (r % 2) * 40 for r in range(requests)]   # 3 or 83: positions 702 and 782
        window = 200                                                # tokens 503.. and 583..
        k, v = torch.randn(prefix, 1, d, generator=g), torch.randn(prefix, 1, d, generator=g)
        v[560] = bad
        pages = -(-prefix // 64)
        cache = sa.Kv4Cache.empty(pages + 2 * requests, 1, d, page_size=64, device=dev)
        slots = torch.arange(prefix, dtype=torch.int32)
        cache.append(k.to(dev), v.to(dev), slots.to(dev))
        tables = pages + 2 * torch.arange(requests, dtype=torch.int32)[:, None] + torch.tensor([0, 1], dtype=torch.int32)
        ks, vs = [], []
        for r, x in enumerate(lengths):
            j = torch.arange(x)
            s = tables[r][j // 64] * 64 + (j % 64).to(torch.int32)
            cache.append(torch.randn(x, 1, d, generator=g).to(dev), torch.randn(x, 1, d, generator=g).to(dev), s.to(dev))
            a, b = cache.read(s.to(dev))
            ks.append(a.cpu().double())
            vs.append(b.cpu().double())
        pk, pv = (x.cpu().double() for x in cache.read(slots.to(dev)))
        q = _queries(requests, 1, 2, d, dtype, 3, dev)
        out = cache.attend_shared(q, torch.arange(pages, dtype=torch.int32, device=dev), _i32([prefix], dev), tables.to(dev),
                                  _i32(lengths, dev), window=window)
        for r, x in enumerate(lengths):
            if x == 3:
                assert not torch.isfinite(out[r]).any() if bad != bad or dtype == F16 else (out[r].abs() > 1e10).any()
                continue
            sees = R.visible(1, prefix + x, window, 0)
            ref, spread, score, _ = L.attend(q[r].cpu().double(), torch.cat([pk, ks[r]]), torch.nan_to_num(torch.cat([pv, vs[r]])),
                                             sees, 0.125)
            _close(out[r], ref, spread, score, d, prefix + x, P_SHARED[dtype])


def test_shared_prefix_of_nothing_is_attend(dev):
    cache, tables, lens, _, _ = _filled(dev, [0, 50, 3], 2, 64, 16, F32, 5)
    q = _queries(2, 1, 4, 64, BF16, 1, dev)
    want = cache.attend(q, tables[1:], lens[1:])
    _one_step(cache.attend_shared(q, tables[0], lens[:1], tables[1:], lens[1:]), want)
    _one_step(cache.attend_shared(q, tables[0, :0], lens[:1], tables[1:], lens[1:]), want)
    empty = cache.attend_shared(q[:0], tables[0], lens[:1], tables[:0], lens[:0])
    assert empty.shape == (0, 1, 4, 64)


# ------------------------------------------------------------ selected pages

PAGES = [
    # lengths, heads, kv heads, n, d, page, count
    ([1], 1, 1, 1, 64, 16, 1),
    ([1, 0, 5, 16, 17, 300], 4, 2, 1, 128, 16, 4),
    ([40, 1000, 257], 8, 1, 2, 128, 64, 5),
    ([333, 64, 2, 0], 6, 2, 3, 64, 16, 7),
    ([700, 31], 24, 1, 1, 32, 64, 20),
    ([515, 90], 24, 1, 2, 256, 16, 9),
    ([100, 129], 6, 3, 5, 80, 32, 1),
    ([77, 50], 2, 2, 1, 7, 16, 3),
    ([9000], 8, 2, 1, 128, 64, 100),
]


def _lists(lengths, n, h, page, count, seed):
    g = R.rng(seed)
    out = torch.full((len(lengths), n, h, count), -1, dtype=torch.int32)
    for r, x in enumerate(lengths):
        for i in range(n):
            for j in range(h):
                rows = -(-x // page)   # some of them behind the query
                take = min(rows, count)
                out[r, i, j, :take] = torch.randperm(rows, generator=g)[:take].sort().values.to(torch.int32)
    return out


@TYPES
@pytest.mark.parametrize("case", range(len(PAGES)))
def test_attend_pages_matches_definition(case, dtype, dev):
    lengths, heads, h, n, d, page, count = PAGES[case]
    cache, tables, lens, ks, vs = _filled(dev, lengths, h, d, page, F32, case)
    q = _queries(len(lengths), n, heads, d, dtype, case, dev)
    pages = _lists(lengths, n, h, page, count, case)
    out = cache.attend_pages(q, tables, lens, pages.to(dev))
    assert out.shape == q.shape and out.dtype == dtype
    for r, x in enumerate(lengths):
        sees = torch.zeros(h, n, x, dtype=torch.bool)
        for i in range(n):
            for j in range(h):
                for w in pages[r, i, j].tolist():
                    if w >= 0:
                        sees[j, i, w * page:(w + 1) * page] = True
        sees &= R.visible(n, x, None, 0)
        ref, spread, score, _ = L.attend(q[r].cpu().double(), ks[r], vs[r], sees, 1 / math.sqrt(d))
        _close(out[r], ref, spread, score, d, count * page, P_HALF[dtype])
    if n == 1:
        assert torch.equal(cache.attend_pages(q[:, 0], tables, lens, pages[:, 0].to(dev)), out[:, 0])


def test_attend_pages_all_and_none(dev):
    lengths = [150, 40, 0]
    cache, tables, lens, _, _ = _filled(dev, lengths, 2, 64, 16, F32, 1)
    q = _queries(3, 1, 4, 64, BF16, 1, dev)
    every = torch.arange(10, dtype=torch.int32).expand(3, 1, 2, 10).contiguous()
    every = torch.where(every < torch.tensor([10, 3, 0])[:, None, None, None], every, -1).to(torch.int32).to(dev)
    _one_step(cache.attend_pages(q, tables, lens, every), cache.attend(q, tables, lens))
    none = torch.full((3, 1, 2, 4), -1, dtype=torch.int32, device=dev)
    assert (cache.attend_pages(q, tables, lens, none) == 0).all()
    assert (cache.attend_pages(q, tables, lens, none[..., :0]) == 0).all()


@pytest.mark.parametrize("bad", [[2, 2, 3], [0, 5, 3], [1, 4, 99], [1, -7, 4], [1, -1, 4]])
def test_attend_pages_lists_out_of_order(bad, dev):
    """Entries from the first bad one on count as none, and it is reported; behind a -1 nobody looks."""
    cache, tables, lens, _, _ = _filled(dev, [90], 1, 64, 16, F32, 1)
    q = _queries(1, 1, 2, 64, BF16, 1, dev)
    at = next(i for i in range(1, 3) if bad[i] <= bad[i - 1] or bad[i] >= tables.shape[1])
    good = cache.attend_pages(q, tables, lens, _i32([[[bad[:at]]]], dev))
    if bad[at] == -1:
        assert torch.equal(cache.attend_pages(q, tables, lens, _i32([[[bad]]], dev)), good)
    else:
        with pytest.raises(ValueError, match="list of pages"):
            cache.attend_pages(q, tables, lens, _i32([[[bad]]], dev))


# ------------------------------------------------------- bounds and selection

@pytest.mark.parametrize("d,page", [(1, 16), (31, 16), (32, 64), (64, 32), (80, 128), (128, 64), (200, 16), (256, 256)])
def test_bounds_are_the_definition(d, page, dev):
    lengths, h = [1, 0, page, page + 1, 5 * page - 3], 3
    cache, tables, lens, ks, _ = _filled(dev, lengths, h, d, page, F32, d)
    dp = cache.padded_dim(d)
    for new in ([1, 1, 1, 1, 1], [0, 3, page, 2, 2 * page + 1], [1, 0, page, page + 1, 10 ** 6], [-5, 0, 0, 0, 0]):
        bounds = cache.page_bounds().fill_(7.0)
        cache.update_page_bounds(bounds, tables, lens, _i32(new, dev))
        want = torch.full(bounds.shape, 7.0, dtype=BF16)
        for r, x in enumerate(lengths):
            first = max(0, x - max(new[r], 0))
            for w in range(first // page, -(-x // page) if first < x else 0):
                for j in range(h):
                    want[tables[r, w], j] = L.bounds(ks[r][w * page:(w + 1) * page, j], d, dp)
        assert torch.equal(bounds.cpu(), want)


def test_bounds_of_nan_and_bad_pages(dev):
    cache, tables, lens, _, _ = _filled(dev, [40], 1, 64, 16, F32, 3)
    cache.k_params[tables[0, 1], 0, 3] = float("nan")
    bounds = cache.page_bounds()
    cache.update_page_bounds(bounds, tables, lens, lens)
    assert torch.isnan(bounds[tables[0, 1]]).all() and torch.isfinite(bounds[tables[0, 0]]).all()
    tables[0, 0] = -1
    with pytest.raises(ValueError, match="outside the cache"):
        cache.update_page_bounds(bounds, tables, lens, lens)


SELECT = [
    # lengths, heads, kv heads, n, d, page, count, first, last
    ([1], 1, 1, 1, 64, 16, 1, 1, 0),
    ([1, 0, 5, 16, 17, 300], 4, 2, 1, 128, 16, 4, 1, 1),
    ([40, 3000, 257], 8, 1, 1, 128, 16, 20, 0, 0),
    ([333, 64, 2, 0], 6, 2, 3, 64, 16, 7, 2, 3),
    ([700, 31], 24, 1, 1, 32, 16, 6, 3, 3),
    ([515, 90], 24, 1, 2, 256, 16, 9, 1, 1),
    ([100, 129], 6, 3, 5, 80, 32, 2, 0, 1),
    ([77, 50], 2, 2, 1, 7, 16, 3, 1, 1),
    ([12000], 8, 2, 1, 64, 16, 300, 1, 2),
    ([5000] * 3, 8, 4, 2, 128, 16, 31, 1, 1),
]


@TYPES
@pytest.mark.parametrize("case", range(len(SELECT)))
def test_select_is_the_definition(case, dtype, dev):
    lengths, heads, h, n, d, page, count, first, last = SELECT[case]
    cache, tables, lens, _, _ = _filled(dev, lengths, h, d, page, F32, case)
    bounds = cache.page_bounds()
    cache.update_page_bounds(bounds, tables, lens, lens)
    wide = _queries(len(lengths), n, heads + 3, d, dtype, case, dev)
    q = wide[:, :, 2:2 + heads]
    got = cache.select_pages(q, bounds, tables, lens, count=count, first=first, last=last)
    assert got.dtype == torch.int32 and got.shape == (len(lengths), n, h, count)
    b, qc = bounds.cpu().double()[..., :d], q.cpu().double()
    per = heads // h
    for r, x in enumerate(lengths):
        rows = -(-x // page)
        at = b[tables[r, :rows].long().cpu()]
        for i in range(n):
            own = x - (n - 1 - i)
            for j in range(h):
                want = L.select(qc[r, i, j * per:(j + 1) * per], at[:, j, 0], at[:, j, 1], max(0, -(-own // page)), count,
                                first, last)
                assert got[r, i, j].tolist() == want, (r, i, j)
    if n == 1:
        assert torch.equal(cache.select_pages(q[:, 0], bounds, tables, lens, count=count, first=first, last=last), got[:, 0])


@pytest.mark.parametrize("pages", [40, 3000])
def test_select_ties_go_to_the_lowest_page(pages, dev):
    """Equal bounds on many pages, signed zeros, and a NaN page that comes first."""
    h, d, page = 1, 32, 16
    cache = sa.Kv4Cache.empty(pages, h, d, page_size=page, device=dev)
    bounds = cache.page_bounds()
    level = torch.tensor([0.0, 1.0, -2.0, 1.0])[torch.arange(pages) % 4]
    bounds[:, 0, 0] = bounds[:, 0, 1] = level[:, None].to(dev).to(BF16)
    tables = torch.arange(pages, dtype=torch.int32, device=dev)[None]
    lens = _i32([pages * page], dev)
    q = torch.ones(1, 1, d, dtype=BF16, device=dev)
    for count in (2, 5, 20, pages // 2 + 1, pages - 1):
        for qs in (q, -q, torch.zeros_like(q), -torch.zeros_like(q)):
            got = cache.select_pages(qs, bounds, tables, lens, count=count, first=0, last=0)[0, 0].tolist()
            value = (level * qs.float().cpu().sum()).tolist()
            assert got == sorted(sorted(range(pages), key=lambda w: (-value[w], w))[:count])
    bounds[7] = float("nan")
    assert cache.select_pages(q, bounds, tables, lens, count=2, first=0, last=0)[0, 0].tolist() == [1, 7]


def test_select_reports_bad_pages(dev):
    cache, tables, lens, _, _ = _filled(dev, [200], 1, 64, 16, F32, 3)
    q = _queries(1, 1, 2, 64, BF16, 1, dev)
    tables[0, 4] = 10 ** 6
    with pytest.raises(ValueError, match="outside the cache"):
        cache.select_pages(q, cache.page_bounds(), tables, lens, count=3)
    with pytest.raises(NotImplementedError, match="24576"):
        cache.select_pages(q, cache.page_bounds(), tables.new_zeros((1, 24577)), lens, count=3)


# ------------------------------------------------------ weights and eviction

WEIGH = [
    # lengths, heads, kv heads, n, d, page, window, sinks
    ([1], 1, 1, 1, 64, 16, None, 0),
    ([1, 0, 5, 16, 17, 300], 4, 2, 1, 128, 16, None, 0),
    ([40, 1000, 257], 32, 4, 1, 128, 128, 100, 4),
    ([333, 64, 2, 0], 6, 2, 3, 64, 16, 50, 1),
    ([700, 31], 20, 1, 3, 32, 64, None, 0),
    ([515, 90], 24, 1, 2, 256, 16, 200, 130),
    ([100, 129], 9, 3, 5, 80, 32, 33, 2),
    ([77, 50], 2, 2, 1, 7, 16, 20, 3),
    ([9000, 4100], 8, 2, 1, 128, 64, None, 0),
]


@TYPES
@pytest.mark.parametrize("case", range(len(WEIGH)))
def test_weights_match_definition(case, dtype, dev):
    lengths, heads, h, n, d, page, window, sinks = WEIGH[case]
    cache, tables, lens, ks, vs = _filled(dev, lengths, h, d, page, F32, case)
    q = _queries(len(lengths), n, heads, d, dtype, case, dev)
    weights = cache.token_weights()
    before = torch.rand(weights.shape, generator=R.rng(case))
    weights.copy_(before)
    out = cache.attend(q, tables, lens, window=window, sinks=sinks, weights=weights)
    want, bound = before.double(), torch.zeros(before.shape, dtype=torch.float64)
    for r, x in enumerate(lengths):
        ref, spread, score, p = L.attend(q[r].cpu().double(), ks[r], vs[r], R.visible(n, x, window, sinks), 1 / math.sqrt(d))
        _close(out[r], ref, spread, score, d, x, P_HALF[dtype])
        # a probability's error as in attention_bound (K is centred for all types: a span of 4), and the additions'
        rel = 2 * (d + 2) * 2.0 ** -24 * 4 * score[..., 0].T[:, :, None] + 6 * 2.0 ** -22 + x * 2.0 ** -23 if x else 0
        j = torch.arange(x)
        at = tables[r].cpu().long()[j // page], j % page
        # [heads, n, m] -> [m, kv heads]
        for to, add in ((want, p), (bound, p * rel)):
            to[at[0], :, at[1]] += add.reshape(h, heads // h, n, x).sum((1, 2)).T
    bound += (n * heads // h + 1) * 2.0 ** -24 * want
    assert ((weights.cpu().double() - want).abs() <= bound).all()
    again = before.to(dev)
    assert torch.equal(cache.attend(q, tables, lens, window=window, sinks=sinks, weights=again), out)
    assert torch.equal(again, weights)


def test_weights_of_hidden_tokens_stay(dev):
    """NaN behind the window reaches no weight; slots of nobody stay as they are."""
    cache, tables, lens, _, _ = _filled(dev, [100, 60], 1, 64, 16, F32, 4)
    q = _queries(2, 1, 2, 64, F16, 1, dev)
    cache.k_params[tables[0, 1]] = float("nan")   # tokens 16..31
    weights = cache.token_weights().fill_(-3.0)
    cache.attend(q, tables, lens, window=20, sinks=3, weights=weights)
    seen = torch.zeros(weights.shape, dtype=torch.bool)
    for r, x in enumerate([100, 60]):
        mine = torch.zeros(weights.shape, dtype=torch.bool)
        for t in list(range(3)) + list(range(x - 20, x)):
            mine[tables[r, t // 16], 0, t % 16] = True
        # two heads, each of weight 1: 23 weights added to -3, each rounded by 2^-23 at most
        assert abs((weights.cpu()[mine].double() + 3).sum() - 2.0) < 1e-5
        seen |= mine
    assert (weights.cpu()[~seen] == -3.0).all() and (weights.cpu()[seen] > -3.0).all()


def test_reset_weights(dev):
    cache = sa.Kv4Cache.empty(4, 3, 64, page_size=16, device=dev)
    weights = cache.token_weights().fill_(5.0)
    cache.reset_weights(weights, _i32([3, -1, 63, 16], dev))
    want = torch.full((4, 3, 16), 5.0)
    want[0, :, 3] = want[3, :, 15] = want[1, :, 0] = 0.0
    assert torch.equal(weights.cpu(), want)
    with pytest.raises(ValueError, match="slot of token 1"):
        cache.reset_weights(weights, _i32([0, 64], dev))


EVICT = [
    # lengths, kv heads, d, page, keep, limit, first, last
    ([5], 1, 64, 16, 3, 3, 0, 0),
    ([5], 1, 64, 16, 5, 5, 0, 0),
    ([100, 0, 33, 34, 16, 300], 2, 128, 16, 33, 33, 1, 5),
    ([100, 0, 33, 90, 16, 300], 3, 80, 32, 33, 90, 4, 29),
    ([1000, 1500, 700], 2, 64, 64, 600, 700, 4, 100),
    ([257, 2], 4, 256, 16, 1, 1, 0, 1),
    ([257, 2], 4, 31, 16, 2, 200, 1, 0),
    ([3000], 1, 128, 256, 130, 256, 0, 0),
    ([90] * 40, 1, 32, 16, 70, 70, 2, 3),
    ([25600, 26000], 1, 32, 256, 24900, 25599, 10, 300),   # more than stand in shared memory
]


def _free(cache, tables, dev):
    """A free list of the pages that no request holds, with room for all."""
    pages = [p for p in range(cache.num_pages) if p not in set(tables.flatten().tolist())]
    return pages + [-9] * (cache.num_pages - len(pages)), len(pages)


@pytest.mark.parametrize("kind", ["random", "ties", "special"])
@pytest.mark.parametrize("case", range(len(EVICT)))
def test_evict_is_the_definition(case, kind, dev):
    lengths, h, d, page, keep, limit, first, last = EVICT[case]
    cache, tables, lens, ks, vs = _filled(dev, lengths, h, d, page, F32, case)
    g = R.rng(case)
    weights = torch.exp(2 * torch.randn(cache.num_pages, h, page, generator=g))
    if kind == "ties":
        weights = weights.round().clamp(max=2)
    if kind == "special":   # signs, signed zeros, infinities and NaN
        weights = torch.tensor([0.0, -0.0, -1.0, math.inf, -math.inf, math.nan, 1e-42, 3.0])[
            torch.randint(0, 8, weights.shape, generator=g)]
    was, tables_was = weights.clone(), tables.cpu()
    free, count = _free(cache, tables, dev)
    w, lens_d, free_d, count_d = weights.to(dev), lens.clone(), _i32(free, dev), _i32([count], dev)
    kept, dropped = cache.evict(w, lens_d, tables, free_d, count_d, keep=keep, limit=limit, first=first, last=last)
    over = [x > limit for x in lengths]
    assert lens_d.tolist() == [keep if o else x for o, x in zip(over, lengths)]
    assert dropped.tolist() == [x - keep if o else 0 for o, x in zip(over, lengths)]
    w = w.cpu()
    pages_seen = set()
    for r, x in enumerate(lengths):
        rows = -(-x // page)
        stays = -(-keep // page) if over[r] else rows
        assert tables[r].tolist() == tables_was[r, :stays].tolist() + [-1] * (tables.shape[1] - stays)
        if over[r]:
            free[count:count + rows - stays] = tables_was[r, stays:rows].tolist()
            count += rows - stays
        slots = lambda n: (tables_was[r].long()[torch.arange(n) // page], torch.arange(n) % page)  # noqa: E731
        for j in range(h):
            mine = was[slots(x)[0], j, slots(x)[1]] if x else torch.zeros(0)
            stay = L.keep_of(mine.tolist(), keep, first, last) if over[r] else list(range(min(x, keep)))
            assert kept[r, j].tolist() == stay + [-1] * (keep - len(stay))
            if not over[r]:
                stay = list(range(x))
            at, off = slots(len(stay))
            assert torch.equal(torch.nan_to_num(w[at, j, off], nan=-77.0), torch.nan_to_num(mine[stay], nan=-77.0))
            if over[r]:
                cells = rows * page
                at, off = slots(cells)
                assert (w[at, j, off][keep:] == 0).all()
            if stay:
                at, off = slots(len(stay))
                k, v = cache.read((at * page + off).to(torch.int32).to(dev))
                assert torch.equal(k[:, j].cpu().double(), ks[r][stay, j]) and torch.equal(v[:, j].cpu().double(), vs[r][stay, j])
        pages_seen |= set(tables_was[r, :rows].tolist())
    assert free_d.tolist() == free and count_d.tolist() == [count]
    others = [p for p in range(cache.num_pages) if p not in pages_seen]
    assert torch.equal(torch.nan_to_num(w[others], nan=-77.0), torch.nan_to_num(was[others], nan=-77.0))


def test_evict_leaves_other_slots_of_a_page(dev):
    """Codes of the slots behind the last kept token stay what they were, within a word of values too."""
    cache, tables, lens, _, _ = _filled(dev, [40], 1, 64, 16, F32, 1)
    before = cache.v_codes.clone(), cache.k_codes.clone()
    cache.evict(cache.token_weights(), lens, tables, _i32([0] * 9, dev), _i32([0], dev), keep=17)
    page = tables[0, 1].item()
    rest = torch.arange(1, 16) + page * 16
    assert torch.equal(R.v_rows(cache.v_codes, rest, 64), R.v_rows(before[0], rest, 64))
    assert torch.equal(R.k_rows(cache.k_codes, rest, 64), R.k_rows(before[1], rest, 64))


def test_evict_reports(dev):
    cache, tables, lens, _, _ = _filled(dev, [40], 1, 64, 16, F32, 1)
    w = cache.token_weights()
    with pytest.raises(ValueError, match="more than the output holds"):   # a free list without room
        cache.evict(w, lens.clone(), tables.clone(), _i32([0] * 6, dev), _i32([5], dev), keep=3)
    with pytest.raises(ValueError, match="outside the cache"):   # a list of fewer pages than the cache has
        cache.evict(w, lens.clone(), torch.where(tables >= 0, 4, tables), _i32([0] * 3, dev), _i32([0], dev), keep=3)
    bad = tables.clone()
    bad[0, 1] = 10 ** 6
    with pytest.raises(ValueError, match="outside the cache"):
        cache.evict(w, lens.clone(), bad, _i32([0] * 9, dev), _i32([0], dev), keep=3)
    with pytest.raises(ValueError, match="longer than its row"):
        cache.evict(w, lens.clone() + 100, tables.clone(), _i32([0] * 9, dev), _i32([0], dev), keep=3)


# --------------------------------------------------------------- used together

def _serve(dev, steps, graph):
    """A batch behind a shared prompt: each step appends a token, attends over the pages it selects, over
    prompt and own tokens, and with weights; then evicts.  Captured or not."""
    g = R.rng(11)
    r, h, heads, d, page, width = 3, 2, 4, 64, 16, 8
    cache = sa.Kv4Cache.empty(64, h, d, page_size=page, device=dev)
    prompt = torch.arange(100, dtype=torch.int32, device=dev)   # pages 0..6
    kp, vp = (torch.randn(100, h, d, generator=g).to(dev) for _ in range(2))
    cache.append(kp, vp, prompt)
    prefix_table, prefix_length = torch.arange(7, dtype=torch.int32, device=dev), _i32([100], dev)
    lengths, tables = _i32([0] * r, dev), torch.full((r, width), -1, dtype=torch.int32, device=dev)
    free, count = torch.arange(63, -1, -1, dtype=torch.int32, device=dev), _i32([57], dev)
    new, weights, bounds = _i32([1] * r, dev), cache.token_weights().fill_(9.0), cache.page_bounds()
    xs = torch.randn(steps, r, heads + 2 * h, d, generator=g).to(dev)
    x = xs[0].clone()

    def step():
        q, k, v = x[:, :heads], x[:, heads:heads + h], x[:, heads + h:]
        plan = sa.plan_kv_pages(lengths, new, tables, free, count, page_size=page, per_request=1)
        cache.append(k, v, plan.slots)
        cache.reset_weights(weights, plan.slots)
        lengths.copy_(plan.lengths)
        count.copy_(plan.free_count)
        shared = cache.attend_shared(q, prefix_table, prefix_length, tables, lengths, window=90, sinks=4)
        cache.update_page_bounds(bounds, tables, lengths, new)
        pages = cache.select_pages(q, bounds, tables, lengths, count=2)
        sparse = cache.attend_pages(q, tables, lengths, pages)
        own = cache.attend(q, tables, lengths, weights=weights)
        kept, dropped = cache.evict(weights, lengths, tables, free, count, keep=30, limit=37, first=2, last=8)
        cache.update_page_bounds(bounds, tables, lengths, lengths)
        return shared, pages, sparse, own, kept, dropped

    outs = []
    if graph:
        saved = [t.clone() for t in (cache.k_codes, cache.k_params, cache.v_codes, cache.v_params, lengths, tables, free, count,
                                     weights, bounds)]
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            step()   # loads the code
        torch.cuda.synchronize()
        for t, s in zip((cache.k_codes, cache.k_params, cache.v_codes, cache.v_params, lengths, tables, free, count, weights,
                         bounds), saved):
            t.copy_(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
    for i in range(steps):
        x.copy_(xs[i])
        if graph:
            graph.replay()
        else:
            got = step()
        outs.append([t.clone() for t in got] + [lengths.clone(), count.clone(), weights[tables.long().clamp(min=0)].clone()])
    sa.check_serving_status(dev)
    return outs


def test_a_run_of_all_of_them_captured_and_not(dev):
    a, b = _serve(dev, 60, False), _serve(dev, 60, True)
    for x, y in zip(a, b):
        for s, t in zip(x, y):
            assert torch.equal(s, t)
    assert a[-1][6].tolist() == [a[-1][6][0].item()] * 3 and max(o[5].max().item() for o in a) == 8
    # weights of a token and head: its queries' of every step since it came, each of weight 1 in all
    assert all(torch.isfinite(t.float()).all() for o in a for t in o)


def test_sparse_attention_with_every_page_is_attend(dev):
    cache, tables, lens, _, _ = _filled(dev, [500, 90, 17], 2, 128, 16, F32, 9)
    q = _queries(3, 1, 8, 128, BF16, 2, dev)
    bounds = cache.page_bounds()
    cache.update_page_bounds(bounds, tables, lens, lens)
    pages = cache.select_pages(q, bounds, tables, lens, count=32)
    _one_step(cache.attend_pages(q, tables, lens, pages), cache.attend(q, tables, lens))


def test_calls_on_other_streams_with_workspaces(dev):
    """Two streams at once, each with its own tensors and workspaces."""
    sets = []
    for seed in range(2):
        cache, tables, lens, _, _ = _filled(dev, [700] + [40 + seed] * 50, 2, 64, 16, F32, seed)
        sets.append((cache, tables, lens, _queries(50, 1, 4, 64, BF16, seed, dev)))
    want = []
    for cache, tables, lens, q in sets:
        w = cache.token_weights()
        want.append((cache.attend_shared(q, tables[0], lens[:1], tables[1:], lens[1:]),
                     cache.attend(q, tables[1:], lens[1:], weights=w), w))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for i, (stream, (cache, tables, lens, q)) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(stream):
                w = cache.token_weights()
                got[i].append((cache.attend_shared(q, tables[0], lens[:1], tables[1:], lens[1:]),
                               cache.attend(q, tables[1:], lens[1:], weights=w), w))
    torch.cuda.synchronize()
    for i in range(2):
        for y in got[i]:
            assert all(torch.equal(s, t) for s, t in zip(want[i], y))
