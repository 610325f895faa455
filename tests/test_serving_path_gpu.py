"""Page plans, norm + rotation, and the serving operators run together as
StreamingWindowAttention does."""

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


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


# ---------------------------------------------------------------- page plans

def _state(lengths, page, width, seed, spare=0, extra=None):
    g = R.rng(seed)
    held = [-(-x // page) for x in lengths]
    pages = sum(held) + (extra if extra is not None else len(lengths) * width) + spare
    order = torch.randperm(pages, generator=g).tolist()
    tables, at = [], 0
    for x in held:
        tables.append(order[at:at + x] + [-1] * (width - x))
        at += x
    free = order[at:] + order[:at]
    return tables, free, pages - at


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("requests", [1, 2, 31, 255, 256, 257, 700])
def test_plan_matches_token_by_token(page, requests, dev):
    g = R.rng(page + requests)
    lengths = torch.randint(0, 200, (requests,), generator=g).tolist()
    new = torch.randint(0, 90, (requests,), generator=g).tolist()
    new[0] = 0 if requests > 1 else new[0]
    width = -(-300 // page)
    tables, free, count = _state(lengths, page, width, requests)
    want = R.plan(lengths, new, tables, free, count, page)
    t = _i32(tables, dev)
    for cap in (sum(new), sum(new) + 333):
        got = sa.plan_kv_pages(_i32(lengths, dev), _i32(new, dev), t, _i32(free, dev), _i32([count], dev), page_size=page,
                               max_tokens=cap)
        pad = [-1] * (cap - sum(new))
        assert got.lengths.tolist() == want[0] and got.offsets.tolist() == want[1]
        assert got.positions.tolist() == want[2] + pad and got.slots.tolist() == want[3] + pad
        assert got.tables is t and t.tolist() == want[4] and got.free_count.tolist() == [want[5]]


def test_plan_one_long_request_and_many_empty(dev):
    lengths, new = [0] * 50 + [7] + [0] * 50, [0] * 50 + [50000] + [0] * 49 + [1]
    tables, free, count = _state(lengths, 16, 3200, 1, extra=4000)
    want = R.plan(lengths, new, tables, free, count, 16)
    got = sa.plan_kv_pages(_i32(lengths, dev), _i32(new, dev), _i32(tables, dev), _i32(free, dev), _i32([count], dev),
                           page_size=16, max_tokens=50001)
    assert got.slots.tolist() == want[3] and got.positions.tolist() == want[2] and got.tables.tolist() == want[4]
    assert got.free_count.tolist() == [want[5]]


def test_plan_per_request_rows(dev):
    lengths, new = [15, 16, 0, 31, 40], [2, 1, 0, 3, 0]
    tables, free, count = _state(lengths, 16, 4, 3)
    want = R.plan(lengths, new, tables, free, count, 16)
    got = sa.plan_kv_pages(_i32(lengths, dev), _i32(new, dev), _i32(tables, dev), _i32(free, dev), _i32([count], dev),
                           page_size=16, per_request=3)
    slots, positions, at = [], [], 0
    for x in new:
        slots += want[3][at:at + x] + [-1] * (3 - x)
        positions += want[2][at:at + x] + [-1] * (3 - x)
        at += x
    assert got.slots.tolist() == slots and got.positions.tolist() == positions
    assert got.tables.tolist() == want[4] and got.offsets.tolist() == want[1] and got.lengths.tolist() == want[0]


def test_plan_large_batch(dev):
    """Above the shared memory that needs no opt-in."""
    requests = 16384
    g = R.rng(4)
    lengths = torch.randint(0, 30, (requests,), generator=g).tolist()
    new = torch.randint(0, 4, (requests,), generator=g).tolist()
    tables, free, count = _state(lengths, 16, 3, 4)
    want = R.plan(lengths, new, tables, free, count, 16)
    got = sa.plan_kv_pages(_i32(lengths, dev), _i32(new, dev), _i32(tables, dev), _i32(free, dev), _i32([count], dev),
                           page_size=16, max_tokens=sum(new))
    assert got.slots.tolist() == want[3] and got.tables.tolist() == want[4] and got.offsets.tolist() == want[1]


def test_plan_shortages_are_reported(dev):
    lengths, new = [10, 20], [30, 30]
    tables, free, count = _state(lengths, 16, 4, 5, extra=2)
    args = lambda t, c: (_i32(lengths, dev), _i32(new, dev), t, _i32(free, dev), _i32([c], dev))  # noqa: E731
    with pytest.raises(ValueError, match="pages wanted"):      # 4 wanted, 2 free
        sa.plan_kv_pages(*args(_i32(tables, dev), count), page_size=16, max_tokens=60)
    t = _i32([r[:2] for r in tables], dev)
    with pytest.raises(ValueError, match="longer than its row|pages wanted"):
        sa.plan_kv_pages(*args(t, count), page_size=16, max_tokens=60)
    tables, free, count = _state(lengths, 16, 4, 5)
    with pytest.raises(ValueError, match="more than the output holds"):
        sa.plan_kv_pages(*args(_i32(tables, dev), count), page_size=16, max_tokens=59)
    with pytest.raises(ValueError, match="more than the output holds"):
        sa.plan_kv_pages(*args(_i32(tables, dev), count), page_size=16, per_request=29)
    bad = [10 ** 6] * len(free)
    with pytest.raises(ValueError, match="outside the cache"):
        sa.plan_kv_pages(_i32(lengths, dev), _i32(new, dev), _i32(tables, dev), _i32(bad, dev), _i32([count], dev),
                         page_size=16, max_tokens=60)
    sa.check_serving_status(dev)


def test_plan_empty(dev):
    z = torch.zeros(0, dtype=torch.int32, device=dev)
    p = sa.plan_kv_pages(z, z, z.reshape(0, 4), z, _i32([0], dev), page_size=16, max_tokens=5)
    assert p.slots.tolist() == [-1] * 5 and p.offsets.tolist() == [0] and p.free_count.tolist() == [0]
    p = sa.plan_kv_pages(_i32([3], dev), _i32([0], dev), _i32([[0]], dev), _i32([0], dev), _i32([0], dev), page_size=16,
                         max_tokens=0)
    assert p.lengths.tolist() == [3] and p.slots.numel() == 0


def test_release_returns_every_page_once(dev):
    lengths = [100, 0, 17, 4000, 16]
    tables, free, count = _state(lengths, 16, 260, 6, extra=10)
    t, f, c, n = _i32(tables, dev), _i32(free, dev), _i32([count], dev), _i32(lengths, dev)
    drop = torch.tensor([True, True, False, True, False], device=dev)
    sa.release_kv_pages(n, t, drop, f, c, page_size=16)
    back = [p for r in (0, 3) for p in tables[r] if p >= 0]
    assert c.tolist() == [count + len(back)]
    assert f.tolist()[:count + len(back)] == free[:count] + back
    assert n.tolist() == [0, 0, 17, 0, 16]
    assert t[2].tolist() == tables[2] and t[4].tolist() == tables[4] and (t[[0, 1, 3]] == -1).all()
    sa.release_kv_pages(n, t, drop, f, c, page_size=16)     # again: nothing is left to return
    assert c.tolist() == [count + len(back)]


def test_plan_and_release_refusals(dev):
    n, t, f, c = _i32([1], dev), _i32([[0, -1]], dev), _i32([1, 0], dev), _i32([1], dev)
    with pytest.raises(ValueError, match="page_size"):
        sa.plan_kv_pages(n, n, t, f, c, page_size=10, max_tokens=1)
    with pytest.raises(ValueError, match="either max_tokens or per_request"):
        sa.plan_kv_pages(n, n, t, f, c, page_size=16)
    with pytest.raises(ValueError, match="per_request must be positive"):
        sa.plan_kv_pages(n, n, t, f, c, page_size=16, per_request=0)
    with pytest.raises(ValueError, match="lengths must have shape"):
        sa.plan_kv_pages(_i32([1, 2], dev), n, t, f, c, page_size=16, max_tokens=1)
    with pytest.raises(ValueError, match="tables must be contiguous"):
        sa.plan_kv_pages(n, n, t.long(), f, c, page_size=16, max_tokens=1)
    with pytest.raises(ValueError, match="CUDA tensors"):
        sa.plan_kv_pages(n.cpu(), n, t, f, c, page_size=16, max_tokens=1)
    with pytest.raises(ValueError, match="drop must be bool"):
        sa.release_kv_pages(n, t, n, f, c, page_size=16)
    with pytest.raises(NotImplementedError, match="requests"):
        big = torch.zeros(16385, dtype=torch.int32, device=dev)
        sa.plan_kv_pages(big, big, big[:, None].contiguous(), f, c, page_size=16, max_tokens=1)


# ---------------------------------------------------------- norm and rotation

def _rotary_bound(ref, dtype):
    """float32: the mean of d squares (d / 2 + 3 roundings at most, by pairs or
    lanes fewer), root, divide, two products, then two products and a sum of
    values no larger than the pair's norm, cos and sin off by 2^-22; one rounding
    of the output.  The pair's norm is bounded by the row's largest |y| * sqrt(2)."""
    top = ref.abs().amax(-1, keepdim=True) * 2 ** 0.5
    return R.HALF[dtype] * ref.abs() + (24 * 2.0 ** -24 + 4 * 2.0 ** -22) * top + (2.0 ** -25 if dtype == F16 else 1e-37)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,half,interleaved", [(128, 64, False), (128, 64, True), (64, 32, False), (256, 128, False), (128, 32, False),
                                                (128, 16, True), (80, 40, False), (96, 20, False), (7, 3, False), (33, 16, True), (64, 0, False),
                                                (2, 1, False), (1, 0, False), (72, 36, True)])
@pytest.mark.parametrize("weights", [True, False])
def test_rotary_matches_definition(dtype, d, half, interleaved, weights, dev):
    g = R.rng(d + half)
    t, h, hkv = 37, 5, 2
    q, k = (torch.randn(t, x, d, generator=g).to(dtype) * 3 for x in (h, hkv))
    positions = torch.randint(0, 2 ** 31 - 1, (t,), generator=g)
    positions[:8] = torch.tensor([0, 1, 2, 4095, 131071, 10 ** 6, 10 ** 9, 2 ** 31 - 1])
    wq, wk = ((1 + 0.3 * torch.randn(d, generator=g)).to(dtype) for _ in range(2)) if weights else (None, None)
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))
    to = lambda x: None if x is None else x.to(dev)  # noqa: E731
    got = sa.qk_norm_rotary(q.to(dev), k.to(dev), positions.to(torch.int32).to(dev), to(wq), to(wk), freq.to(dev), eps=1e-5,
                            interleaved=interleaved)
    for x, w, y in ((q, wq, got[0]), (k, wk, got[1])):
        ref = R.rotary(x.double(), positions, w, freq, 1e-5, interleaved)
        assert y.dtype == dtype and y.is_contiguous()
        # an angle of position p is p frequency, exact in float64 to 2^-53 of it: 2^31 2^-53 is far below the bound
        R.assert_close(y, ref, _rotary_bound(ref, dtype))


@pytest.mark.parametrize("d", [128, 64, 50])
def test_rotary_strides_in_place_and_padding(d, dev):
    g = R.rng(d)
    qkv = torch.randn(20, 8, d, generator=g).to(BF16).to(dev)
    positions = torch.arange(20, dtype=torch.int32)
    positions[[2, 19]] = -1
    freq = sa.rotary_frequencies(d, device=dev)
    q, k = qkv[:, :4], qkv[:, 4:6]
    pd = positions.to(dev)
    a, b = sa.qk_norm_rotary(q, k, pd, None, None, freq)
    gone = positions < 0
    assert (a[gone.to(dev)] == 0).all() and (b[gone.to(dev)] == 0).all()
    ref = R.rotary(q.cpu().double(), positions, None, freq.cpu(), 1e-6, False)
    R.assert_close(a[~gone.to(dev)], ref[~gone], _rotary_bound(ref[~gone], BF16))
    same = qkv.clone()
    sa.qk_norm_rotary(same[:, :4], same[:, 4:6], pd, None, None, freq, out=(same[:, :4], same[:, 4:6]))
    assert torch.equal(same[~gone.to(dev)][:, :4], a[~gone.to(dev)]) and torch.equal(same[~gone.to(dev)][:, 4:6], b[~gone.to(dev)])
    assert torch.equal(same[gone.to(dev)], qkv[gone.to(dev)]) and torch.equal(same[:, 6:], qkv[:, 6:])
    shifted = torch.randn(20 * 6 * d + 1, generator=g).to(BF16).to(dev)[1:].view(20, 6, d)      # off 16-byte borders
    x, _ = sa.qk_norm_rotary(shifted[:, :4], shifted[:, 4:], pd, None, None, freq)
    y, _ = sa.qk_norm_rotary(shifted[:, :4].contiguous().clone(), shifted[:, 4:].contiguous(), pd, None, None, freq)
    assert torch.equal(x, y)


def test_rotary_zero_rows_and_extremes(dev):
    q = torch.zeros(3, 2, 64, device=dev)
    q[1] = 1e18
    q[2, 0, 0] = float("nan")
    pos = torch.arange(3, dtype=torch.int32, device=dev)
    a, b = sa.qk_norm_rotary(q, q[:, :1], pos, None, None, sa.rotary_frequencies(64, device=dev))
    assert (a[0] == 0).all() and torch.isfinite(a[1]).all() and torch.isnan(a[2, 0]).any() and (a[2, 1] == 0).all()
    e = sa.qk_norm_rotary(q[:0], q[:0], pos[:0], None, None, sa.rotary_frequencies(64, device=dev))
    assert e[0].shape == (0, 2, 64)


def test_rotary_refusals(dev):
    q, pos, f = torch.zeros(3, 2, 64, device=dev), torch.zeros(3, dtype=torch.int32, device=dev), sa.rotary_frequencies(64, device=dev)
    for bad, match in ((lambda: sa.qk_norm_rotary(q, q[:2], pos, None, None, f), r"\[T,H,D\]"),
                       (lambda: sa.qk_norm_rotary(q, q, pos.long(), None, None, f), "int32"),
                       (lambda: sa.qk_norm_rotary(q, q, pos, None, None, f.float()), "float64"),
                       (lambda: sa.qk_norm_rotary(q[..., :62], q[..., :62], pos, None, None, f), "2 R <= 62"),
                       (lambda: sa.qk_norm_rotary(q, q, pos, q[0, 0, :3], None, f), "q_weight"),
                       (lambda: sa.qk_norm_rotary(q, q, pos, q[0, 0].half(), None, f), "one dtype"),
                       (lambda: sa.qk_norm_rotary(q, q, pos, None, None, f, out=(q, q.half())), "out must match"),
                       (lambda: sa.rotary_frequencies(7), "even")):
        with pytest.raises(ValueError, match=match):
            bad()


# ------------------------------------------------------------------ together

class _Plain:
    """The same layer in float64, request by request: the cache holds what the 4-bit definition gives."""

    def __init__(self, layer):
        self.l, self.k, self.v = layer, {}, {}

    def rotate(self, x, positions, w):
        return R.rotary(x.double(), positions, w, self.l.frequencies.cpu(), self.l.eps, self.l.interleaved)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("graph", [False, True])
def test_prompt_and_decode_through_the_cache(dtype, graph, dev):
    """Prompts of a ragged batch, decode steps, a request that ends and its slot
    reused: each step's output against float64 attention over the rows that the
    steps before put in, which are read back from the cache."""
    heads, hkv, d, window, sinks, page = 8, 2, 64, 40, 3, 16
    g = R.rng(77)
    wq, wk = ((1 + 0.1 * torch.randn(d, generator=g)).to(dtype).to(dev) for _ in range(2))
    layer = sa.StreamingWindowAttention(heads, hkv, d, max_requests=4, max_length=160, window=window, sinks=sinks, q_weight=wq,
                                        k_weight=wk, page_size=page, device=dev)
    mk = lambda t: tuple(torch.randn(t, x, d, generator=g).to(dtype).to(dev) for x in (heads, hkv, hkv))  # noqa: E731
    lens = [0, 0, 0, 0]

    def held(r):
        j = torch.arange(lens[r], device=dev)
        slots = (layer.tables[r].long()[j // page] * page + j % page).to(torch.int32)
        return tuple(x.double().cpu() for x in layer.cache.read(slots))

    def prompt(new):
        t = sum(new)
        q, k, v = mk(t + 5)
        out = layer.prefill(q, k, v, _i32(new, dev))
        assert (out[t:] == 0).all()
        at = 0
        for r, x in enumerate(new):
            if not x:
                continue
            assert lens[r] == 0
            lens[r] = x
            pos = torch.arange(x)
            rows = slice(at, at + x)
            # the prompt's attention runs over the rotated keys as rounded to the inputs' type
            qr, kr = sa.qk_norm_rotary(q[rows], k[rows], pos.to(torch.int32).to(dev), wq, wk, layer.frequencies)
            ref, spread, score = R.attention(*(y.double().cpu().repeat_interleave(heads // y.shape[1], 1).transpose(0, 1)
                                               for y in (qr, kr, v[rows])), R.visible(x, x, window, sinks), d ** -0.5)
            p_half = 0.0 if dtype == F32 else R.HALF[dtype]
            R.assert_close(out[rows].transpose(0, 1), ref, R.attention_bound(ref, spread, score, d, x, dtype, p_half))
            # and the cache holds the quantised rows
            hk, hv = held(r)
            for y, z in ((kr, hk), (v[rows], hv)):
                assert torch.equal(R.value_of(*R.quantise(y.cpu().double())).double(), z)
            at += x

    prompt([37, 0, 16, 101])
    assert layer.lengths.tolist() == lens
    captured = None
    for step in range(6):
        q, k, v = mk(4)
        if graph:
            if captured is None:
                state = [x.clone() for x in (layer.lengths, layer.tables, layer.free_count)]
                ins = tuple(x.clone() for x in (q, k, v))
                side = torch.cuda.Stream(dev)
                side.wait_stream(torch.cuda.current_stream(dev))
                with torch.cuda.stream(side):
                    layer.decode(*ins)
                torch.cuda.current_stream(dev).wait_stream(side)
                for x, y in zip((layer.lengths, layer.tables, layer.free_count), state):
                    x.copy_(y)
                captured = torch.cuda.CUDAGraph()
                with torch.cuda.graph(captured):
                    out_g = layer.decode(*ins)
            for x, y in zip(ins, (q, k, v)):
                x.copy_(y)
            captured.replay()
            out = out_g.clone()
        else:
            out = layer.decode(q, k, v)
        torch.cuda.synchronize()
        for r in range(4):
            if lens[r] == 0:
                assert (out[r] == 0).all()
                continue
            lens[r] += 1
            hk, hv = held(r)
            qr, _ = sa.qk_norm_rotary(q[r:r + 1], k[r:r + 1], _i32([lens[r] - 1], dev), wq, wk, layer.frequencies)
            kk, vv = (y.repeat_interleave(heads // hkv, 1).transpose(0, 1) for y in (hk, hv))
            ref, spread, score = R.attention(qr.double().cpu().transpose(0, 1), kk, vv, R.visible(1, lens[r], window, sinks), d ** -0.5)
            R.assert_close(out[r:r + 1].transpose(0, 1), ref,
                           R.attention_bound(ref, spread, R.code_span(dtype) * score, d, lens[r], dtype, 0.0 if dtype == F32 else 2.0 ** -16))
        assert layer.lengths.tolist() == lens
        if step == 2:
            before = layer.free_count.item()
            layer.release(torch.tensor([False, False, True, True], device=dev))
            assert layer.free_count.item() == before + sum(-(-lens[r] // page) for r in (2, 3))
            lens[2] = lens[3] = 0
            prompt([0, 9, 0, 64])
    sa.check_serving_status(dev)


def test_layer_refusals(dev):
    with pytest.raises(ValueError, match="multiple of the key heads"):
        sa.StreamingWindowAttention(3, 2, 64, max_requests=1, max_length=10, device=dev)
    with pytest.raises(ValueError, match="page_size"):
        sa.StreamingWindowAttention(2, 2, 64, max_requests=1, max_length=10, page_size=0, device=dev)
    layer = sa.StreamingWindowAttention(2, 2, 64, max_requests=2, max_length=10, device=dev)
    x = torch.zeros(3, 2, 64, device=dev)
    with pytest.raises(ValueError, match="one row for each"):
        layer.decode(x, x, x)
    with pytest.raises(ValueError, match="q, k, v must be"):
        layer.prefill(x, x[:2], x, _i32([1, 1], dev))
