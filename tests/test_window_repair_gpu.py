"""Windowed attention where a value that is not finite stands in a tile, seen or
hidden, and where the scale is zero."""

import os

import pytest
import torch

import serving_ref as R
import streaming_attention_b200 as sa
from streaming_attention_b200 import _lib, fast

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return torch.device("cuda:0")


def _make(g, dev, dtype, *shape):
    return torch.randn(*shape, generator=g, device=dev).to(dtype)


def _bound(q, k, v, window, sinks, scale, dtype):
    """The float64 result of one [H,N,D] sequence and its bound, on the GPU."""
    sees = R.visible(q.shape[1], k.shape[1], window, sinks).to(q.device)
    per = q.shape[0] // k.shape[0]
    kd, vd = (x.double().repeat_interleave(per, 0) for x in (k, v))
    ref, spread, score = R.attention(q.double(), kd, vd, sees, scale)
    keys = min(k.shape[1], (window or k.shape[1]) + sinks)
    half = 0.0 if dtype == F32 else R.HALF[dtype]
    return ref.cpu(), R.attention_bound(ref, spread, score, q.shape[-1], keys, dtype, half).cpu()


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_scale_of_zero(dtype, dev):
    """The mean of the visible values; 16-bit types take the CUDA cores' kernel for it, bit for bit."""
    g = torch.Generator(dev).manual_seed(1)
    q, k, v = (_make(g, dev, dtype, 1, 2, 300, 64) for _ in range(3))
    out = sa.sliding_window_attention(q, k, v, window=70, sinks=3, scale=0.0)
    R.assert_close(out[0], *_bound(q[0], k[0], v[0], 70, 3, 0.0, dtype))
    if dtype != F32:
        old = os.environ.get("SA_FORCE_SIMT")
        os.environ["SA_FORCE_SIMT"] = "1"
        try:
            plain = sa.sliding_window_attention(q, k, v, window=70, sinks=3, scale=0.0)
        finally:
            if old is None:
                del os.environ["SA_FORCE_SIMT"]
            else:
                os.environ["SA_FORCE_SIMT"] = old
        assert torch.equal(out, plain)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("n,m", [(700, 700), (3, 5000)], ids=["whole", "split"])
def test_one_bad_column_is_one_bad_column(dtype, bad, n, m, dev):
    """A value that is not finite in one column of one key: the queries that see it
    have it there and nowhere else; the others are as if it were not there."""
    g = torch.Generator(dev).manual_seed(2)
    q, k, v = (_make(g, dev, dtype, 1, 4, n, 64), *(_make(g, dev, dtype, 1, 2, m, 64) for _ in range(2)))
    for at, window, sinks in ((2, 150, 4), (5, 150, 4), (m - 130, 150, 4), (m - 2, None, 0)):
        w = v.clone()
        w[:, :, at, 37] = bad
        out = sa.sliding_window_attention(q, k, w, window=window, sinks=sinks)
        ref, bound = _bound(q[0], k[0], v[0], window, sinks, 0.125, dtype)
        sees = R.visible(n, m, window, sinks)[:, at]
        cols = torch.arange(64) != 37
        R.assert_close(out[0][..., cols.to(dev)], ref[..., cols], bound[..., cols])
        R.assert_close(out[0][:, ~sees.to(dev)], ref[:, ~sees], bound[:, ~sees])
        hit = out[0, :, sees.to(dev), 37].float().cpu()
        assert (torch.isnan(hit) if bad != bad else hit == bad).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_keys_that_are_not_finite_make_their_readers_nan(dtype, dev):
    g = torch.Generator(dev).manual_seed(3)
    q, k, v = (_make(g, dev, dtype, 1, 2, 400, 128 if dtype != F32 else 64) for _ in range(3))
    ref, bound = _bound(q[0], k[0], v[0], 60, 0, q.shape[-1] ** -0.5, dtype)
    for bad in (float("nan"), float("inf"), float("-inf")):
        w = k.clone()
        w[:, :, 200, 5] = bad
        w[:, :, 200, 6] = -bad
        q[..., 5:7] = 1.0
        ref, bound = _bound(q[0], k[0], v[0], 60, 0, q.shape[-1] ** -0.5, dtype)
        out = sa.sliding_window_attention(q, w, v, window=60, sinks=0)[0]
        assert torch.isnan(out[:, 200:260]).all()
        for rows in (slice(0, 200), slice(260, None)):
            R.assert_close(out[:, rows], ref[:, rows], bound[:, rows])


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_repairs_of_any_length_end_no_wait(dtype, dev):
    """A hidden NaN beside the first tokens makes every row of the call one to repair,
    each over two thousand keys.  That takes many times the limit that the waits
    have here, and the CTA's other warps wait behind it: all rows come out."""
    g = torch.Generator(dev).manual_seed(4)
    heads, n, m, window = 320, 256, 2400, 2000
    q, k, v = _make(g, dev, dtype, 1, heads, n, 64), *(_make(g, dev, dtype, 1, heads, m, 64) for _ in range(2))
    bad = v.clone()
    bad[:, :, 5] = float("nan")
    sa.sliding_window_attention(q, k, v, window=window, sinks=4)
    lib = _lib.load()
    try:
        _lib.check(lib.sa_set_wait_limit_ns(1000000), "limit")
        out = sa.sliding_window_attention(q, k, bad, window=window, sinks=4)
        torch.cuda.synchronize(dev)
    finally:
        lib.sa_set_wait_limit_ns(0)
    for h in (0, 147, 148, 319):
        R.assert_close(out[0, h:h + 1], *_bound(q[0, h:h + 1], k[0, h:h + 1], v[0, h:h + 1], window, 4, 0.125, dtype))
    assert torch.isfinite(out).all()


def test_a_bad_first_token_of_a_long_prompt(dev):
    """Every query sees it, so every row is NaN, and that is found at once."""
    g = torch.Generator(dev).manual_seed(5)
    q, k, v = (_make(g, dev, BF16, 1, h, 16384, 128) for h in (8, 2, 2))
    k[:, :, 0], v[:, :, 0] = float("nan"), float("nan")
    assert torch.isnan(sa.sliding_window_attention(q, k, v, window=None)).all()
    assert torch.isnan(sa.sliding_window_attention(q, k, v, window=512, sinks=1)).all()


# ------------------------------------------------- offsets out of order or range

@pytest.fixture
def unchecked(monkeypatch):
    """Calls as they are without SA_CHECK_STATUS: nothing raises until somebody asks."""
    monkeypatch.setattr(fast, "_CHECK_STATUS", False)


def _fill_pool(dev, nbytes):
    """What the allocator hands out next is not zero."""
    x = torch.full((nbytes,), 0x3C, dtype=torch.uint8, device=dev)
    del x


BAD_OFFSETS = [
    # cu_q, cu_k of 40 rows; which rows of a new result are zero
    ([0, 10, 30, 55], [0, 10, 30, 40], range(30, 40)),
    ([0, 10, 30, 40], [0, 10, 50, 40], range(10, 40)),
    ([-4, 10, 30, 36], [0, 10, 30, 40], [*range(10), *range(36, 40)]),
    ([0, 10, 20, 5], [0, 10, 20, 40], range(20, 40)),
    ([8, 50, 60, 70], [0, 10, 20, 30], range(40)),
    ([3, 12, 12, 12], [0, 41, 41, 41], range(40)),
    ([30, 40, 40, 20], [0, 40, 40, 40], range(30)),
]


@pytest.mark.parametrize("dtype,d", [(F32, 64), (F16, 64), (BF16, 128), (BF16, 200)])
@pytest.mark.parametrize("case", range(len(BAD_OFFSETS)))
def test_every_row_of_a_new_result_is_written(case, dtype, d, unchecked, dev):
    """Requests with bad offsets are skipped and reported, the others right, and no
    row of a new result is what the allocator gave; a given one keeps its rows."""
    cu_q, cu_k, zero = BAD_OFFSETS[case]
    g = torch.Generator(dev).manual_seed(case)
    q, k, v = (_make(g, dev, dtype, 40, h, d) for h in (4, 2, 2))
    to = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    f = lambda **kw: sa.sliding_window_attention_packed(q, k, v, to(cu_q), to(cu_k), window=7, sinks=1, **kw)  # noqa: E731
    _fill_pool(dev, q.numel() * q.element_size())
    out = f()
    with pytest.raises(ValueError, match="offsets of request"):
        sa.check_serving_status(dev)
    given = f(out=torch.full_like(q, 7.0))
    with pytest.raises(ValueError, match="offsets of request"):
        sa.check_serving_status(dev)
    zero = torch.tensor(sorted(zero), dtype=torch.long, device=dev)
    assert (out[zero] == 0).all() and (given[zero] == 7.0).all()
    seen = set(zero.tolist())
    for a, b, c, e in zip(cu_q, cu_q[1:], cu_k, cu_k[1:]):
        if 0 <= a <= b <= 40 and 0 <= c <= e <= 40 and b > a:
            ref, bound = _bound(q[a:b].transpose(0, 1), k[c:e].transpose(0, 1), v[c:e].transpose(0, 1), 7, 1, d ** -0.5, dtype)
            for x in (out, given):
                R.assert_close(x[a:b].transpose(0, 1), ref, bound)
            seen |= set(range(a, b))
    assert seen == set(range(40))


@pytest.mark.parametrize("dtype,d", [(F32, 64), (BF16, 64)], ids=["f32", "bf16"])
def test_offsets_that_step_back_over_many_tiles(dtype, d, unchecked, dev):
    """Requests behind a step back take tiles of the long one before it."""
    n = 4000
    cu = torch.tensor([0, n, 50, 51, 52, 53, 54, 54, 60], dtype=torch.int32, device=dev)
    g = torch.Generator(dev).manual_seed(8)
    q, k, v = (_make(g, dev, dtype, n, 1, d) for _ in range(3))
    _fill_pool(dev, q.numel() * q.element_size())
    out = sa.sliding_window_attention_packed(q, k, v, cu, cu, window=30)[:, 0]
    with pytest.raises(ValueError, match="offsets of request"):
        sa.check_serving_status(dev)
    ref, bound = (x[0].to(dev) for x in _bound(*(x.transpose(0, 1) for x in (q, k, v)), 30, 0, d ** -0.5, dtype))
    right = ((out.double() - ref).abs() <= bound).all(1)
    right[50:60] = True          # claimed twice
    assert (right | (out == 0).all(1)).all() and torch.isfinite(out).all() and right.sum() > 100


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_prefill_with_fewer_rows_than_new_tokens(dtype, unchecked, dev):
    """The request that the rows end in, and those behind it, are reported; their rows are zero."""
    layer = sa.StreamingWindowAttention(4, 2, 64, max_requests=3, max_length=64, window=20, sinks=1, page_size=16, device=dev)
    g = torch.Generator(dev).manual_seed(9)
    q, k, v = (_make(g, dev, dtype, 40, h, 64) for h in (4, 2, 2))
    _fill_pool(dev, q.numel() * q.element_size())
    out = layer.prefill(q, k, v, torch.tensor([10, 35, 20], dtype=torch.int32, device=dev))
    with pytest.raises(ValueError):
        sa.check_serving_status(dev)
    assert (out[10:] == 0).all() and torch.isfinite(out).all() and (out[:10] != 0).any()


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype,d", [(F32, 64), (F32, 128), (F16, 64), (BF16, 128), (BF16, 200)])
def test_a_row_that_sees_nothing_but_nan_is_nan(dtype, d, packed, dev):
    """Whatever kernel takes it: a key that is NaN, alone in a window, or before all the others that a row sees."""
    g = torch.Generator(dev).manual_seed(6)
    q, k, v = (_make(g, dev, dtype, 1, 2, 300, d) for _ in range(3))
    k[:, :, 0], k[:, :, 200] = float("nan"), float("nan")
    cu = torch.tensor([0, 300], dtype=torch.int32, device=dev)
    rows = lambda x: x[0].transpose(0, 1).contiguous()  # noqa: E731
    for window, sinks in ((1, 0), (1, 1), (64, 0), (None, 0)):
        if packed:
            out = sa.sliding_window_attention_packed(rows(q), rows(k), rows(v), cu, cu, window=window, sinks=sinks)
            out = out.transpose(0, 1)[None]
        else:
            out = sa.sliding_window_attention(q, k, v, window=window, sinks=sinks)
        sees = R.visible(300, 300, window, sinks)
        bad = (sees[:, 0] | sees[:, 200]).to(dev)
        assert torch.isnan(out[:, :, bad]).all() and torch.isfinite(out[:, :, ~bad]).all()


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("h,hkv,n,m,window,sinks", [(80, 80, 130, 40000, None, 0), (80, 80, 130, 40000, 36000, 4), (32, 8, 512, 70000, None, 0)],
                         ids=["whole", "window", "split"])
def test_chains_that_are_folded(h, hkv, n, m, window, sinks, dtype, dev):
    """Over 32768 keys and more: rising scores late in a chain, which all that was
    folded is scaled down for, and values that are not finite, seen and hidden."""
    g = torch.Generator(dev).manual_seed(7)
    q, k, v = _make(g, dev, dtype, 1, h, n, 64), *(_make(g, dev, dtype, 1, hkv, m, 64) for _ in range(2))
    k[:, :, m - 3000] *= 4
    k[:, 0, 34000:] += q[:, 0, :1] * 0.5        # the first query's scores rise by 16 there
    w = v.clone()
    w[:, :, 20000, 3] = float("inf")
    w[:, :, m - 1] = float("nan")                # seen by the last query alone
    if sinks:
        w[:, :, 6] = float("nan")                # hidden, beside the first tokens
    for values, cols in ((v, slice(None)), (w, torch.arange(64) != 3)):
        out = sa.sliding_window_attention(q, k, values, window=window, sinks=sinks)
        for at in (0, h - 1):
            y = at // (h // hkv)
            ref, bound = _bound(q[0, at:at + 1], k[0, y:y + 1], v[0, y:y + 1], window, sinks, 0.125, dtype)
            rows = slice(0, n if values is v else n - 1)
            R.assert_close(out[0, at:at + 1, rows][..., cols], ref[:, rows][..., cols], bound[:, rows][..., cols])
        if values is w:
            assert torch.isnan(out[:, :, n - 1]).all() and (out[:, :, :n - 1, 3] == float("inf")).all()
