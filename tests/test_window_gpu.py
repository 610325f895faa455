"""Windowed attention with first tokens that stay visible, against the float64
masked softmax: element by element, within the roundings that the kernels make
(serving_ref.attention_bound; with 16-bit inputs the probabilities are rounded
once to the inputs' type, with float32 inputs not at all)."""

import math

import pytest
import torch

import serving_ref as R
import streaming_attention_b200 as sa

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return torch.device("cuda:0")


def _p_half(dtype):
    return 0.0 if dtype == F32 else R.HALF[dtype]


def _make(shape, dtype, g, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def _check(q, k, v, out, window, sinks, scale=None):
    """q [B,H,N,D], k / v [B,Hkv,M,*] and out [B,H,N,Dv], any device."""
    per = q.shape[1] // k.shape[1]
    sees = R.visible(q.shape[2], k.shape[2], window, sinks)
    sc = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    for b in range(q.shape[0]):
        qd = q[b].cpu().double()
        kd, vd = (x[b].cpu().double().repeat_interleave(per, 0) for x in (k, v))
        ref, spread, score = R.attention(qd, kd, vd, sees, sc)
        keys = min(k.shape[2], (window or k.shape[2]) + sinks)
        R.assert_close(out[b], ref, R.attention_bound(ref, spread, score, q.shape[-1], keys, out.dtype, _p_half(out.dtype)))


SHAPES = [
    # b, h, hkv, n, m, d, dv, window, sinks
    (1, 1, 1, 1, 1, 64, 64, 1, 0),
    (2, 4, 2, 1, 200, 128, 128, 64, 4),
    (1, 8, 1, 3, 513, 64, 64, 130, 1),
    (2, 3, 3, 127, 127, 32, 32, 16, 0),
    (1, 4, 4, 128, 128, 64, 64, None, 0),
    (1, 4, 2, 129, 129, 128, 128, 128, 2),
    (1, 2, 1, 255, 400, 128, 64, 100, 130),
    (1, 2, 2, 257, 257, 64, 128, 1, 1),
    (1, 6, 2, 300, 301, 80, 80, 33, 7),
    (2, 2, 1, 64, 700, 96, 96, 250, 64),
    (1, 2, 1, 700, 700, 128, 128, 200, 129),
    (1, 2, 2, 385, 640, 64, 64, 5000, 3),
    (1, 1, 1, 513, 513, 128, 128, 512, 0),
    (1, 2, 2, 40, 90, 7, 5, 11, 2),
    (1, 2, 1, 65, 65, 33, 127, 20, 0),
    (1, 2, 2, 70, 150, 256, 256, 64, 5),
    (1, 2, 1, 130, 260, 192, 100, 65, 40),
    (1, 16, 2, 2, 1500, 128, 128, 1000, 20),
    (1, 2, 1, 1, 4100, 128, 128, None, 0),          # few queries, many keys: the keys are split
    (2, 4, 4, 3, 4211, 64, 96, 3900, 300),
    (1, 8, 2, 70, 4000, 80, 33, None, 0),
    (3, 1, 1, 40, 4700, 48, 48, 3300, 1000),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=["-".join(map(str, s)) for s in SHAPES])
def test_window_matches_definition(shape, dtype, dev):
    b, h, hkv, n, m, d, dv, window, sinks = shape
    g = R.rng(n * 31 + m + d)
    q = _make((b, h, n, d), dtype, g, 1.5)
    k, v = _make((b, hkv, m, d), dtype, g), _make((b, hkv, m, dv), dtype, g)
    out = sa.sliding_window_attention(q.to(dev), k.to(dev), v.to(dev), window=window, sinks=sinks)
    assert out.dtype == dtype and out.shape == (b, h, n, dv) and out.is_contiguous()
    _check(q, k, v, out, window, sinks)


@pytest.mark.parametrize("n", [1, 2, 31, 64, 127, 128, 129, 191, 256, 257, 400])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (7, 0), (64, 1), (127, 128), (128, 0), (129, 127), (None, 0)])
def test_window_edges_bf16(n, window, sinks, dev):
    """Tile borders of queries, windows and first tokens."""
    g = R.rng(n * 1000 + (window or 0) * 7 + sinks)
    q, k, v = _make((1, 2, n, 64), BF16, g, 2.0), _make((1, 1, n + 5, 64), BF16, g), _make((1, 1, n + 5, 64), BF16, g)
    _check(q, k, v, sa.sliding_window_attention(q.to(dev), k.to(dev), v.to(dev), window=window, sinks=sinks), window, sinks)


def test_window_single_sequence_and_scale(dev):
    g = R.rng(5)
    q, k, v = _make((150, 64), F16, g), _make((150, 64), F16, g), _make((150, 32), F16, g)
    out = sa.sliding_window_attention(q.to(dev), k.to(dev), v.to(dev), window=40, sinks=2, scale=-0.3)
    _check(q[None, None], k[None, None], v[None, None], out[None, None], 40, 2, -0.3)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_window_equals_full_attention_when_nothing_is_hidden(dtype, dev):
    g = R.rng(6)
    q, k, v = (_make((1, 2, 300, 64), dtype, g).to(dev) for _ in range(3))
    a = sa.sliding_window_attention(q, k, v, window=None)
    assert torch.equal(a, sa.sliding_window_attention(q, k, v, window=300))
    assert torch.equal(a, sa.sliding_window_attention(q, k, v, window=10 ** 9, sinks=10 ** 9))


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 72, 50])
def test_window_strides(dtype, d, dev):
    """[B,N,H,D] tensors seen as [B,H,N,D], slices of one projection, rows that
    start off 16-byte borders, a batch that repeats one sequence, and strides
    that are larger than the rows."""
    g = R.rng(d)
    b, n, h, hkv = 2, 140, 4, 2
    qkv = _make((b, n, h + 2 * hkv, d), dtype, g).to(dev)
    q, k, v = (x.transpose(1, 2) for x in (qkv[:, :, :h], qkv[:, :, h:h + hkv], qkv[:, :, h + hkv:]))
    _check(q, k, v, sa.sliding_window_attention(q, k, v, window=50, sinks=3), 50, 3)
    flat = _make((1 + b * h * n * d,), dtype, g).to(dev)[1:]
    q1 = flat.view(b, h, n, d)
    _check(q1, k, v, sa.sliding_window_attention(q1, k, v, window=50, sinks=3), 50, 3)
    k1, v1 = (x[:1].expand(b, -1, -1, -1) for x in (k, v))
    _check(q, k1, v1, sa.sliding_window_attention(q, k1, v1, window=50, sinks=3), 50, 3)
    wide = _make((b, h, n, d + 3), dtype, g).to(dev)
    q2, k2, v2 = wide[..., :d], wide[:, :hkv, :, 1:d + 1], wide[:, hkv:, :, 3:]
    _check(q2, k2, v2, sa.sliding_window_attention(q2, k2, v2, window=50, sinks=3), 50, 3)
    q3, k3, v3 = (x.transpose(-1, -2).contiguous().transpose(-1, -2) for x in (q, k, v))
    _check(q3, k3, v3, sa.sliding_window_attention(q3, k3, v3, window=50, sinks=3), 50, 3)


PACKED = [
    ([1], [1], 1, 0),
    ([5, 0, 130, 1, 64], [5, 3, 130, 77, 200], 40, 2),
    ([128, 128, 256], [128, 128, 256], 64, 0),
    ([1] * 20, list(range(1, 21)), 6, 1),
    ([300, 1, 129], [301, 900, 129], None, 0),
    ([0, 0, 0], [0, 7, 0], 5, 0),
    ([10, 64], [4, 64], 30, 1),        # more queries than keys: the first ones stand before the first key
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", range(len(PACKED)))
@pytest.mark.parametrize("d,dv", [(64, 64), (128, 128), (40, 24)])
def test_window_packed(case, dtype, d, dv, dev):
    n, m, window, sinks = PACKED[case]
    g = R.rng(case * 100 + d)
    behind = 70
    q = _make((sum(n) + behind, 4, d), dtype, g).to(dev)
    k, v = _make((sum(m) + 9, 2, d), dtype, g).to(dev), _make((sum(m) + 9, 2, dv), dtype, g).to(dev)
    k[sum(m):] = float("nan")
    v[sum(m):] = float("inf")
    cu_q = torch.tensor([0] + n, dtype=torch.int32).cumsum(0).to(torch.int32).to(dev)
    cu_k = torch.tensor([0] + m, dtype=torch.int32).cumsum(0).to(torch.int32).to(dev)
    out = torch.full((q.shape[0], 4, dv), 7.0, dtype=dtype, device=dev)
    got = sa.sliding_window_attention_packed(q, k, v, cu_q, cu_k, window=window, sinks=sinks, out=out)
    assert got is out
    assert (out[sum(n):] == 7.0).all(), "rows behind the last request were written"
    a = c = 0
    for x, y in zip(n, m):
        _check(q[None, a:a + x].transpose(1, 2), k[None, c:c + y].transpose(1, 2), v[None, c:c + y].transpose(1, 2),
               out[None, a:a + x].transpose(1, 2), window, sinks)
        a, c = a + x, c + y
    fresh = sa.sliding_window_attention_packed(q, k, v, cu_q, cu_k, window=window, sinks=sinks)
    assert torch.equal(fresh[:sum(n)], out[:sum(n)]) and (fresh[sum(n):] == 0).all()


def test_window_packed_equals_dense(dev):
    g = R.rng(11)
    q, k, v = (_make((3, 4, 200, 64), BF16, g).to(dev) for _ in range(3))
    dense = sa.sliding_window_attention(q, k, v, window=77, sinks=5)
    rows = lambda x: x.transpose(1, 2).reshape(600, 4, 64).contiguous()  # noqa: E731
    cu = torch.arange(4, dtype=torch.int32, device=dev) * 200
    packed = sa.sliding_window_attention_packed(rows(q), rows(k), rows(v), cu, cu, window=77, sinks=5)
    ref = rows(dense)
    assert (packed.float() - ref.float()).abs().max() <= 2 ** -6 * ref.float().abs().max()


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("d", [64, 128])
def test_window_hidden_keys_do_not_matter(dtype, bad, d, dev):
    """NaN and infinities in keys and values that a query does not see: its result
    stays within the roundings of the definition over what it sees (the rows that
    share a tile with such a value are computed in another way, without rounded
    probabilities, so they need not be the same bits)."""
    g = R.rng(12)
    n, window, sinks = 260, 50, 2
    q, k, v = (_make((1, 2, n, d), dtype, g).to(dev) for _ in range(3))
    k2, v2 = k.clone(), v.clone()
    k2[:, :, 100] = bad          # seen by the queries 100 .. 149 alone
    v2[:, :, 100] = bad
    got = sa.sliding_window_attention(q, k2, v2, window=window, sinks=sinks)
    keep = torch.ones(n, dtype=torch.bool)
    keep[100:150] = False
    ref, spread, score = R.attention(*(x[0].cpu().double() for x in (q, k, v)), R.visible(n, n, window, sinks), d ** -0.5)
    bound = R.attention_bound(ref, spread, score, d, window + sinks, dtype, _p_half(dtype))
    R.assert_close(got[0][:, keep.to(dev)], ref[:, keep], bound[:, keep])
    assert not torch.isfinite(got[:, :, 100:150]).any()


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_window_split_keys_hide_and_repeat(dtype, dev):
    """Few queries over many keys (16-bit types split them over the SMs): hidden NaN
    and infinities, the same bits twice and in a replayed graph, on another stream."""
    g = R.rng(21)
    q, k, v = _make((1, 4, 2, 64), dtype, g, 1.5).to(dev), *(_make((1, 2, 5000, 64), dtype, g).to(dev) for _ in range(2))
    clean = k.clone(), v.clone()
    k[:, :, 4999], v[:, :, 4999] = float("nan"), float("inf")      # seen by the last query alone
    k[:, :, 700], v[:, :, 700] = float("inf"), float("nan")        # by none
    f = lambda: sa.sliding_window_attention(q, k, v, window=4000, sinks=5)  # noqa: E731
    out = f()
    _check(q[:, :, :1], clean[0][:, :, :4999], clean[1][:, :, :4999], out[:, :, :1], 4000, 5)
    assert not torch.isfinite(out[:, :, 1]).any()
    k.copy_(clean[0])
    v.copy_(clean[1])
    first = f()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = f()
    graph.replay()
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        other = f()
    again = f()
    torch.cuda.synchronize()
    assert torch.equal(first, captured) and torch.equal(first, other) and torch.equal(first, again)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_window_running_maximum_moves(dtype, dev):
    """Scores that climb by thousands along the keys, and that fall: the running
    maximum is moved in every tile, or never again."""
    g = R.rng(13)
    n, d = 600, 64
    q = torch.ones(1, 2, n, d).to(dtype)
    ramp = torch.linspace(-30, 30, n)[None, None, :, None]
    k = (ramp * torch.tensor([1.0, -1.0])[None, :, None, None] + 0.05 * torch.randn(1, 2, n, d, generator=g)).to(dtype)
    v = _make((1, 2, n, d), dtype, g)
    out = sa.sliding_window_attention(q.to(dev), k.to(dev), v.to(dev), window=300, sinks=4)
    _check(q, k, v, out, 300, 4)


def test_window_large_magnitudes(dev):
    """Equal scores near the type's largest value, and values near it."""
    for dtype, big in ((F16, 60000.0), (BF16, 3e38), (F32, 3e38)):
        q = torch.zeros(1, 1, 130, 64, dtype=dtype, device=dev)
        k = torch.full((1, 1, 130, 64), big, dtype=dtype, device=dev)
        v = torch.full((1, 1, 130, 64), big / 2, dtype=dtype, device=dev)
        out = sa.sliding_window_attention(q, k, v, window=20, sinks=1)
        # the weights sum to 1 within 2^-8 (their rounding) and the result is rounded once
        assert ((out.double() / (v.double()) - 1).abs() <= 2 * R.HALF[dtype] + 2 ** -16).all()


def test_window_is_deterministic_and_ordered_on_streams(dev):
    g = R.rng(14)
    q, k, v = (_make((2, 4, 500, 128), BF16, g).to(dev) for _ in range(3))
    first = sa.sliding_window_attention(q, k, v, window=200, sinks=4)
    assert torch.equal(first, sa.sliding_window_attention(q, k, v, window=200, sinks=4))
    a, b = torch.cuda.Stream(dev), torch.cuda.Stream(dev)
    outs = []
    for i in range(6):   # two streams at once, inputs made on the stream just before
        with torch.cuda.stream((a, b)[i % 2]):
            (a, b)[i % 2].wait_stream(torch.cuda.default_stream(dev))
            outs.append(sa.sliding_window_attention(q * 1, k * 1, v * 1, window=200, sinks=4))
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)


def test_window_graph_replay(dev):
    g = R.rng(15)
    q, k, v = (_make((1, 4, 300, 64), F16, g).to(dev) for _ in range(3))
    sa.sliding_window_attention(q, k, v, window=100, sinks=1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sa.sliding_window_attention(q, k, v, window=100, sinks=1)
    for seed in (1, 2):
        for x in (q, k, v):
            x.copy_(_make(tuple(x.shape), F16, R.rng(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, sa.sliding_window_attention(q, k, v, window=100, sinks=1))


@pytest.mark.parametrize("dtype,n", [(F32, 20), (F32, 300), (BF16, 20), (BF16, 300)])
def test_window_of_any_size(dtype, n, dev):
    """Windows and first tokens beyond every position are what no window is."""
    g = R.rng(21)
    q, k, v = (_make((1, 2, n, 64), dtype, g).to(dev) for _ in range(3))
    whole = sa.sliding_window_attention(q, k, v, window=None)
    for window, sinks in ((2 ** 32 + 1, 0), (2 ** 62, 2 ** 62), (2 ** 63 + 5, 0), (1, 2 ** 63 - 1), (1, 2 ** 64 + 1)):
        out = sa.sliding_window_attention(q, k, v, window=window, sinks=sinks)
        _check(q.cpu(), k.cpu(), v.cpu(), out, None, 0)
        assert sinks or torch.equal(out, whole)


def test_window_empty(dev):
    z = lambda *s: torch.zeros(*s, device=dev)  # noqa: E731
    assert sa.sliding_window_attention(z(2, 4, 0, 64), z(2, 4, 9, 64), z(2, 4, 9, 64), window=3).shape == (2, 4, 0, 64)
    assert sa.sliding_window_attention(z(0, 4, 5, 64), z(0, 4, 5, 64), z(0, 4, 5, 32), window=3).shape == (0, 4, 5, 32)
    assert sa.sliding_window_attention(z(0, 64), z(0, 64), z(0, 64), window=3).shape == (0, 64)
    cu = torch.zeros(1, dtype=torch.int32, device=dev)
    out = sa.sliding_window_attention_packed(z(3, 2, 64), z(0, 2, 64), z(0, 2, 64), cu, cu, window=3)
    assert out.shape == (3, 2, 64) and (out == 0).all()


def test_window_bad_offsets_are_reported_and_skipped(dev):
    q = torch.ones(10, 2, 64, device=dev, dtype=BF16)
    ok = torch.tensor([0, 4, 10], dtype=torch.int32, device=dev)
    for bad in ([0, 11, 10], [0, 4, 400], [-3, 4, 10], [0, 7, 3]):
        cu = torch.tensor(bad, dtype=torch.int32, device=dev)
        with pytest.raises(ValueError, match="offsets of request"):
            sa.sliding_window_attention_packed(q, q, q, cu, ok, window=4)
        with pytest.raises(ValueError, match="offsets of request"):
            sa.sliding_window_attention_packed(q, q, q, ok, cu, window=4)
    sa.check_serving_status(dev)   # read once, then clear
    assert (sa.sliding_window_attention_packed(q, q, q, ok, ok, window=4) == 1).all()


def test_window_refusals(dev):
    x = torch.zeros(1, 2, 8, 64, device=dev)
    f = sa.sliding_window_attention
    with pytest.raises(ValueError, match="CUDA tensors"):
        f(x.cpu(), x.cpu(), x.cpu(), window=4)
    with pytest.raises(ValueError, match="window must be positive"):
        f(x, x, x, window=0)
    with pytest.raises(ValueError, match="sinks must be non-negative"):
        f(x, x, x, window=4, sinks=-1)
    with pytest.raises(ValueError, match="fewer keys"):
        f(x, x[:, :, :7], x[:, :, :7], window=4)
    with pytest.raises(ValueError, match="multiple of the key heads"):
        f(x[:, :1], x, x, window=4)
    with pytest.raises(ValueError, match="one dtype"):
        f(x, x.half(), x, window=4)
    with pytest.raises(ValueError, match="unsupported dtype"):
        f(x.double(), x.double(), x.double(), window=4)
    with pytest.raises(ValueError, match="head widths"):
        f(torch.zeros(4, 257, device=dev), torch.zeros(4, 257, device=dev), x[0, 0, :4], window=4)
    with pytest.raises(ValueError, match="same head width"):
        f(x, x[..., :32], x, window=4)
    with pytest.raises(ValueError, match="must match k"):
        f(x, x, x[:, :, :7], window=4)
    with pytest.raises(ValueError, match="batch size"):
        f(x, x.expand(2, -1, -1, -1), x.expand(2, -1, -1, -1), window=4)
    p, cu = x[0].transpose(0, 1), torch.tensor([0, 8], dtype=torch.int32, device=dev)
    h = sa.sliding_window_attention_packed
    with pytest.raises(ValueError, match="int32"):
        h(p, p, p, cu.long(), cu, window=4)
    with pytest.raises(ValueError, match="shape"):
        h(p, p, p, cu, cu[:1], window=4)
    with pytest.raises(ValueError, match="out must be"):
        h(p, p, p, cu, cu, window=4, out=torch.zeros(8, 2, 32, device=dev))
