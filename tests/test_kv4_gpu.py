"""The paged 4-bit cache: codes, scales and least values equal the float64
definition bit for bit, what a slot stands for is read back exactly, and
attention over the cache is the float64 masked softmax over those values within
the kernels' roundings (serving_ref.attention_bound; the probabilities keep at
least 16 bits: 2^-16 for their rounding)."""

import math

import pytest
import torch

import serving_ref as R
import streaming_attention_b200 as sa

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
P_HALF = {F32: 0.0, F16: 2.0 ** -16, BF16: 2.0 ** -16}


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return torch.device("cuda:0")


def _check_rows(cache, k, v, slots):
    """The cache's slots hold exactly what the definition gives for k, v [T,H,D]."""
    for x, rows, par in ((k, R.k_rows(cache.k_codes, slots, cache.dim), cache.k_params),
                         (v, R.v_rows(cache.v_codes, slots, cache.dim), cache.v_params)):
        codes, scale, least = R.quantise(x.cpu().double())
        got = R.params(par, slots)
        assert torch.equal(torch.nan_to_num(got[..., :1], nan=-1.0), torch.nan_to_num(scale, nan=-1.0))
        assert torch.equal(torch.nan_to_num(got[..., 1:], nan=-1.0), torch.nan_to_num(least, nan=-1.0))
        fine = torch.isfinite(scale).expand_as(codes)
        assert torch.equal(rows[fine], codes[fine])
    rk, rv = cache.read(slots.to(torch.int32).to(cache.device))
    for x, got in ((k, rk), (v, rv)):
        codes, scale, least = R.quantise(x.cpu().double())
        assert torch.equal(torch.nan_to_num(got.cpu(), nan=-1e30), torch.nan_to_num(R.value_of(codes, scale, least), nan=-1e30))


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [1, 2, 31, 32, 48, 64, 80, 127, 128, 200, 256])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_append_is_the_definition(dtype, d, page, dev):
    g = R.rng(d * 3 + page)
    t, h = 77, 3
    cache = sa.Kv4Cache.empty(6, h, d, page_size=page, device=dev)
    k = (torch.randn(t, h, d, generator=g) * torch.exp(torch.randn(1, 1, d, generator=g))).to(dtype)
    v = (torch.randn(t, h, d, generator=g) + 3 * torch.randn(t, h, 1, generator=g)).to(dtype)
    slots = torch.randperm(6 * page, generator=g)[:t]
    cache.append(k.to(dev), v.to(dev), slots.to(torch.int32).to(dev))
    _check_rows(cache, k, v, slots)


def test_append_borders_and_extremes(dev):
    """Values on the borders between two codes (ties to even), constant rows, rows
    of denormals, of the type's largest values, of mixed signs and far levels."""
    d = 32
    ramp = torch.arange(d, dtype=torch.float64)
    rows = [torch.where(ramp < 30, ramp / 2, torch.where(ramp < 31, torch.zeros(()), torch.full((), 15.0))).double(),
            (ramp - 7.5) / 2, torch.full((d,), 3.7), torch.full((d,), -0.0), ramp * 2.0 ** -133, ramp * 2.0 ** -140,
            (ramp - 16) * 1e37, torch.where(ramp < 1, -3.3e38, 3.3e38).double(), 1e4 + ramp * 1e-3,
            ramp * 2.0 ** -30 + 2.0 ** -40, torch.where(ramp < 1, 1.0, ramp * 1e-9).double(), -ramp ** 4]
    for dtype in (F32, BF16):
        k = torch.stack(rows).to(dtype)[:, None]
        v = -k
        cache = sa.Kv4Cache.empty(1, 1, d, page_size=16, device=dev)
        slots = torch.arange(len(rows))
        cache.append(k.to(dev), v.to(dev), slots.to(torch.int32).to(dev))
        _check_rows(cache, k, v, slots)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("d", [32, 33, 128])
def test_append_rows_of_the_whole_range(dtype, d, dev):
    """Differences of values that float32 cannot hold, scales whose reciprocals it cannot."""
    g = R.rng(d)
    u = torch.rand(40, 1, d, generator=g, dtype=torch.float64) * 2 - 1
    level = torch.cat([torch.full((10,), 3.38e38, dtype=torch.float64), torch.full((10,), 1.6e38, dtype=torch.float64),
                       10.0 ** torch.linspace(-41, -36, 20, dtype=torch.float64)])
    k = (u * level[:, None, None]).to(dtype)
    cache = sa.Kv4Cache.empty(3, 1, d, page_size=16, device=dev)
    slots = torch.arange(40)
    cache.append(k.to(dev), (-k).to(dev), slots.to(torch.int32).to(dev))
    _check_rows(cache, k, -k, slots)


def test_append_many_near_borders(dev):
    """Rows whose quotients sit within float32 rounding of a border."""
    g = R.rng(9)
    t, d = 4096, 128
    scale = torch.rand(t, 1, 1, generator=g) * 3 + 0.01
    steps = torch.randint(0, 30, (t, 1, d), generator=g).float() / 2
    steps[..., 0], steps[..., 1] = 0.0, 15.0
    k = (steps * scale + torch.randn(t, 1, 1, generator=g)).float()
    cache = sa.Kv4Cache.empty(t // 64, 1, d, page_size=64, device=dev)
    slots = torch.arange(t)
    cache.append(k.to(dev), k.to(dev), slots.to(torch.int32).to(dev))
    _check_rows(cache, k, k, slots)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_append_rows_that_are_not_finite_stand_for_nan(bad, dev):
    g = R.rng(10)
    k, v = torch.randn(8, 2, 64, generator=g), torch.randn(8, 2, 64, generator=g)
    k[3, 1, 5] = bad
    v[6, 0, 63] = bad
    cache = sa.Kv4Cache.empty(1, 2, 64, page_size=16, device=dev)
    cache.append(k.to(dev), v.to(dev), torch.arange(8, dtype=torch.int32, device=dev))
    rk, rv = (x.cpu() for x in cache.read(torch.arange(8, dtype=torch.int32, device=dev)))
    assert torch.isnan(rk[3, 1]).all() and torch.isnan(rv[6, 0]).all()
    keep = torch.ones(8, 2, dtype=torch.bool)
    keep[3, 1] = False
    assert torch.isfinite(rk[keep]).all()
    _check_rows(cache, k, v, torch.arange(8))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 50])
def test_append_strides_padding_and_neighbours(dtype, d, dev):
    """Slices of one projection; padded tokens write nothing; the other slots of a page keep what they hold."""
    g = R.rng(d + 1)
    qkv = torch.randn(40, 8, d, generator=g).to(dtype).to(dev)
    k, v = qkv[:, 4:6], qkv[:, 6:8]
    cache = sa.Kv4Cache.empty(4, 2, d, page_size=16, device=dev)
    for t in (cache.k_codes, cache.v_codes):
        t.fill_(0xA5)
    before = cache.k_codes.clone(), cache.v_codes.clone()
    slots = torch.full((40,), -1, dtype=torch.int32)
    slots[:30] = torch.randperm(64, generator=g)[:30].to(torch.int32)
    slots[[3, 17]] = -1
    cache.append(k, v, slots.to(dev))
    held = slots >= 0
    _check_rows(cache, k[held.to(dev)], v[held.to(dev)], slots[held].long())
    others = torch.tensor(sorted(set(range(64)) - set(slots[held].tolist())))
    assert torch.equal(R.k_rows(cache.k_codes, others, cache.dim), R.k_rows(before[0], others, cache.dim))
    assert torch.equal(R.v_rows(cache.v_codes, others, cache.dim), R.v_rows(before[1], others, cache.dim))
    rk, _ = cache.read(slots.to(dev))
    assert (rk[~held.to(dev)] == 0).all()


@pytest.mark.parametrize("tokens", [3, 64, 200])
def test_append_runs_of_slots(tokens, dev):
    """Consecutive slots from any start, as a prompt has them, over a page border; token by token gives the same bytes."""
    g = R.rng(tokens)
    k, v = (torch.randn(tokens, 2, 128, generator=g).to(BF16).to(dev) for _ in range(2))
    for start in (0, 1, 2, 3, 13):
        a, b = (sa.Kv4Cache.empty(16, 2, 128, page_size=16, device=dev) for _ in range(2))
        slots = torch.arange(start, start + tokens, dtype=torch.int32, device=dev)
        a.append(k, v, slots)
        for i in range(tokens):
            b.append(k[i:i + 1], v[i:i + 1], slots[i:i + 1])
        for x, y in zip((a.k_codes, a.v_codes, a.k_params, a.v_params), (b.k_codes, b.v_codes, b.k_params, b.v_params)):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_read_types(dev):
    g = R.rng(3)
    cache = sa.Kv4Cache.empty(2, 2, 96, page_size=32, device=dev)
    k, v = torch.randn(50, 2, 96, generator=g).to(dev), torch.randn(50, 2, 96, generator=g).to(dev)
    slots = torch.arange(50, dtype=torch.int32, device=dev)
    cache.append(k, v, slots)
    full = cache.read(slots)
    for dtype in (F16, BF16):
        for a, b in zip(cache.read(slots, dtype), full):
            assert a.dtype == dtype and torch.equal(a, b.to(dtype))
    assert cache.read(slots[:0])[0].shape == (0, 2, 96)
    cache.append(k[:0], v[:0], slots[:0])


def test_slots_outside_the_cache_are_reported_and_skipped(dev):
    cache = sa.Kv4Cache.empty(2, 1, 32, page_size=16, device=dev)
    x = torch.randn(3, 1, 32, device=dev)
    slots = torch.tensor([0, 32, 1], dtype=torch.int32, device=dev)
    with pytest.raises(ValueError, match="slot of token 1"):
        cache.append(x, x, slots)
    with pytest.raises(ValueError, match="slot of token 1"):
        cache.read(slots)
    _check_rows(cache, x[[0, 2]], x[[0, 2]], torch.tensor([0, 1]))


# ------------------------------------------------------------------ attend

def _filled(dev, lengths, h, d, page, dtype, seed, spare=3):
    """A cache with `lengths` tokens per request in shuffled pages; also the values it stands for."""
    g = R.rng(seed)
    need = [-(-x // page) for x in lengths]
    pages = sum(need) + spare
    width = max(need + [1]) + 1
    order = torch.randperm(pages, generator=g)
    tables = torch.full((len(lengths), width), -1, dtype=torch.int32)
    cache = sa.Kv4Cache.empty(pages, h, d, page_size=page, device=dev)
    # what no request holds is garbage: any code, NaN scales
    cache.k_codes.fill_(0xF7)
    cache.v_codes.fill_(0x7F)
    cache.k_params.fill_(float("nan"))
    cache.v_params.fill_(float("nan"))
    at, ks, vs = 0, [], []
    for r, x in enumerate(lengths):
        tables[r, :need[r]] = order[at:at + need[r]].to(torch.int32)
        at += need[r]
        k, v = (torch.randn(x, h, d, generator=g) for _ in range(2))
        j = torch.arange(x)
        slots = tables[r].long()[j // page] * page + j % page
        cache.append(k.to(dtype).to(dev), v.to(dtype).to(dev), slots.to(torch.int32).to(dev))
        a, b = cache.read(slots.to(torch.int32).to(dev))
        ks.append(a.cpu().double())
        vs.append(b.cpu().double())
    return cache, tables.to(dev), torch.tensor(lengths, dtype=torch.int32, device=dev), ks, vs


def _check_attend(out, q, ks, vs, lengths, window, sinks, scale=None):
    """out, q [R,N,H,D]."""
    n, heads, d = q.shape[1:]
    sc = 1.0 / math.sqrt(d) if scale is None else scale
    for r, x in enumerate(lengths):
        per = heads // ks[r].shape[1] if ks[r].ndim == 3 and ks[r].shape[1] else 1
        k, v = (y.repeat_interleave(per, 1).transpose(0, 1) for y in (ks[r], vs[r]))
        sees = R.visible(n, x, window, sinks)
        ref, spread, score = R.attention(q[r].cpu().double().transpose(0, 1), k, v, sees, sc)
        R.assert_close(out[r].transpose(0, 1), ref,
                       R.attention_bound(ref, spread, R.code_span(out.dtype) * score, d, x, out.dtype, P_HALF[out.dtype]))


ATTEND = [
    # lengths, heads, kv heads, n, d, page, window, sinks
    ([1], 1, 1, 1, 64, 16, None, 0),
    ([1, 0, 5, 16, 17, 300], 4, 2, 1, 128, 16, None, 0),
    ([40, 1000, 257], 8, 1, 1, 128, 64, None, 0),
    ([40, 1000, 257], 32, 4, 1, 128, 128, 100, 4),
    ([2000], 4, 4, 1, 64, 32, 500, 7),
    ([333, 64, 2, 0], 6, 2, 3, 64, 16, 50, 1),
    ([700, 31], 16, 1, 2, 32, 64, None, 0),
    ([515, 90], 24, 1, 2, 256, 16, 200, 130),
    ([100, 129], 6, 3, 5, 80, 32, 33, 2),
    ([77, 50], 2, 2, 1, 7, 16, 20, 3),
    ([260, 9], 5, 1, 1, 127, 256, 1, 1),
    ([150], 12, 4, 4, 200, 64, 64, 0),
    ([9000, 4100], 8, 2, 1, 128, 64, None, 0),
    ([5000], 64, 2, 2, 128, 64, 4096, 4),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_attend_matches_definition(case, dtype, dev):
    lengths, heads, h, n, d, page, window, sinks = ATTEND[case]
    cache, tables, lens, ks, vs = _filled(dev, lengths, h, d, page, F32, case)
    q = (torch.randn(len(lengths), n, heads, d, generator=R.rng(case + 50)) * 1.5).to(dtype).to(dev)
    out = cache.attend(q, tables, lens, window=window, sinks=sinks)
    assert out.shape == q.shape and out.dtype == dtype
    _check_attend(out, q, ks, vs, lengths, window, sinks)
    if n == 1:
        assert torch.equal(cache.attend(q[:, 0], tables, lens, window=window, sinks=sinks), out[:, 0])


@pytest.mark.parametrize("length", list(range(1, 40)) + [63, 64, 65, 127, 128, 129, 511, 512, 513])
def test_attend_lengths(length, dev):
    """Every end within a page and a tile, single request, window and first tokens inside it."""
    cache, tables, lens, ks, vs = _filled(dev, [length], 2, 64, 16, F32, length)
    q = torch.randn(1, 1, 4, 64, generator=R.rng(length)).to(BF16).to(dev)
    for window, sinks in ((None, 0), (9, 2), (16, 17)):
        _check_attend(cache.attend(q, tables, lens, window=window, sinks=sinks), q, ks, vs, [length], window, sinks)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_attend_extreme_scores(dtype, dev):
    """Scores in the thousands that climb along the cache; values far off zero."""
    g = R.rng(8)
    d, x = 64, 900
    cache = sa.Kv4Cache.empty(20, 1, d, page_size=64, device=dev)
    k = torch.linspace(-40, 40, x)[:, None, None] * torch.ones(1, 1, d) + 0.3 * torch.randn(x, 1, d, generator=g)
    v = torch.randn(x, 1, d, generator=g)
    tables = torch.arange(20, dtype=torch.int32, device=dev)[None]
    slots = torch.arange(x, dtype=torch.int32, device=dev)
    cache.append(k.to(dev), v.to(dev), slots)
    ks, vs = (y.cpu().double() for y in cache.read(slots))
    lens = torch.tensor([x], dtype=torch.int32, device=dev)
    for sign in (1.0, -1.0):
        q = (sign * torch.ones(1, 1, 2, d)).to(dtype).to(dev)
        _check_attend(cache.attend(q, tables, lens, window=400, sinks=5), q, [ks], [vs], [x], 400, 5)


def test_attend_large_values_do_not_overflow(dev):
    d = 64
    for dtype, level in ((F16, 3e4), (BF16, 1e30), (F32, 1e30)):
        cache = sa.Kv4Cache.empty(8, 1, d, page_size=16, device=dev)
        k = torch.randn(100, 1, d, generator=R.rng(1)).to(dev)
        v = (torch.randn(100, 1, d, generator=R.rng(2)) * level / 4).to(dev)
        slots = torch.arange(100, dtype=torch.int32, device=dev)
        cache.append(k, v, slots)
        ks, vs = (y.cpu().double() for y in cache.read(slots))
        q = torch.randn(1, 1, 4, d, generator=R.rng(3)).to(dtype).to(dev)
        out = cache.attend(q, torch.arange(8, dtype=torch.int32, device=dev)[None], torch.tensor([100], dtype=torch.int32, device=dev))
        _check_attend(out, q, [ks], [vs], [100], None, 0)


def test_attend_nan_rows_reach_only_queries_that_see_them(dev):
    cache, tables, lens, ks, vs = _filled(dev, [200], 1, 64, 16, F32, 4)
    q = torch.randn(1, 1, 2, 64, generator=R.rng(5)).to(BF16).to(dev)
    clean = cache.attend(q, tables, lens, window=50, sinks=3)
    bad = torch.full((1, 1, 64), float("nan"), device=dev)
    cache.append(bad, bad, (tables[0, 2:3] * 16 + 5))      # position 37: hidden
    assert torch.equal(cache.attend(q, tables, lens, window=50, sinks=3), clean)
    assert torch.isnan(cache.attend(q, tables, lens)).all()


def test_attend_strides_scale_and_streams(dev):
    cache, tables, lens, ks, vs = _filled(dev, [90, 300], 2, 80, 32, F32, 6)
    qkv = torch.randn(2, 2, 10, 81, generator=R.rng(7)).to(F16).to(dev)
    q = qkv[:, :, 1:9, 1:]
    out = cache.attend(q, tables, lens, window=70, sinks=2, scale=0.2)
    _check_attend(out, q, ks, vs, [90, 300], 70, 2, 0.2)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        other = cache.attend(q * 1, tables * 1, lens * 1, window=70, sinks=2, scale=0.2)
    again = cache.attend(q, tables, lens, window=70, sinks=2, scale=0.2)
    torch.cuda.synchronize()
    assert torch.equal(out, other) and torch.equal(out, again)


def test_attend_window_of_any_size(dev):
    """Windows and first tokens beyond every position are what no window is."""
    cache, tables, lens, ks, vs = _filled(dev, [90, 300], 2, 64, 32, F32, 16)
    q = torch.randn(2, 2, 4, 64, generator=R.rng(17)).to(BF16).to(dev)
    whole = cache.attend(q, tables, lens)
    for window, sinks in ((2 ** 32 + 1, 0), (2 ** 63 - 1, 2 ** 63 - 1), (2 ** 64 + 3, 0), (1, 2 ** 63 - 1)):
        out = cache.attend(q, tables, lens, window=window, sinks=sinks)
        _check_attend(out, q, ks, vs, [90, 300], None, 0)
        assert sinks or torch.equal(out, whole)


def test_attend_two_graphs_and_growing_lengths(dev):
    """Two captured calls replayed in turn and at once; lengths and tables change between replays."""
    cache, tables, lens, ks, vs = _filled(dev, [400, 120], 2, 128, 16, F32, 12)
    q = torch.randn(2, 1, 8, 128, generator=R.rng(13)).to(BF16).to(dev)
    cache.attend(q, tables, lens)
    graphs, outs = [], []
    for window in (None, 64):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(cache.attend(q, tables, lens, window=window, sinks=1))
        graphs.append(graph)
    a, b = torch.cuda.Stream(dev), torch.cuda.Stream(dev)
    for sub in ([400, 120], [33, 0], [1, 120]):
        lens.copy_(torch.tensor(sub, dtype=torch.int32))
        torch.cuda.synchronize()
        for s, graph in zip((a, b), graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        cut = lambda xs: [x[:y] for x, y in zip(xs, sub)]  # noqa: E731
        for window, out in zip((None, 64), outs):
            _check_attend(out, q, cut(ks), cut(vs), sub, window, 1)


def test_attend_bad_pages_and_lengths_are_reported(dev):
    cache, tables, lens, ks, vs = _filled(dev, [64], 1, 32, 16, F32, 20)
    q = torch.randn(1, 1, 1, 32, generator=R.rng(21)).to(dev)
    for page in (-1, cache.num_pages, 2 ** 30):
        t = tables.clone()
        t[0, 1] = page
        with pytest.raises(ValueError, match="page .* outside the cache"):
            cache.attend(q, t, lens)
    with pytest.raises(ValueError, match="longer than its row"):
        cache.attend(q, tables[:, :2].contiguous(), lens)
    out = cache.attend(q, tables, torch.full_like(lens, -5))
    assert (out == 0).all()
    _check_attend(cache.attend(q, tables, lens), q, ks, vs, [64], None, 0)


def test_kv4_refusals(dev):
    cache = sa.Kv4Cache.empty(2, 2, 64, page_size=16, device=dev)
    x = torch.zeros(3, 2, 64, device=dev)
    slots = torch.zeros(3, dtype=torch.int32, device=dev)
    tables, lens = torch.zeros(1, 2, dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
    q = torch.zeros(1, 4, 64, device=dev)
    for bad, match in ((lambda: sa.Kv4Cache.empty(2, 2, 64, page_size=24, device=dev), "page_size"),
                       (lambda: sa.Kv4Cache.empty(2, 2, 300, device=dev), "dim must lie"),
                       (lambda: sa.Kv4Cache.empty(0, 2, 64, device=dev), "at least one page"),
                       (lambda: sa.Kv4Cache(cache.k_codes, cache.k_params, cache.v_codes, cache.v_params, 96), "takes 64 bytes"),
                       (lambda: sa.Kv4Cache(cache.k_codes, cache.v_codes, cache.v_codes, cache.v_params, 64), "k_params must be"),
                       (lambda: cache.append(x, x.half(), slots), "one dtype"),
                       (lambda: cache.append(x[:, :1], x[:, :1], slots), "k and v must be"),
                       (lambda: cache.append(x, x, slots.long()), "int32"),
                       (lambda: cache.append(x.cpu(), x.cpu(), slots), "CUDA tensors"),
                       (lambda: cache.append(x.double(), x.double(), slots), "unsupported dtype"),
                       (lambda: cache.read(slots, torch.int8), "unsupported dtype"),
                       (lambda: cache.attend(q[:, :3], tables, lens), "multiple of 2 heads"),
                       (lambda: cache.attend(q[..., :32], tables, lens), "head width 64"),
                       (lambda: cache.attend(q, tables[:, :1].expand(2, 1), lens), "tables must be"),
                       (lambda: cache.attend(q, tables, lens.long()), "int32"),
                       (lambda: cache.attend(q, tables, lens, window=-3), "window must be positive"),
                       (lambda: cache.attend(q, tables, lens, window=3, sinks=-3), "sinks must be"),
                       (lambda: cache.attend(q[0], tables, lens), "q must be")):
        with pytest.raises(ValueError, match=match):
            bad()
