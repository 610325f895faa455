"""How precise the attentions are, as root mean squares over the whole output: an
error that grows with the length of the context shows here long before it passes
the bounds for single elements."""

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


def _rms(x):
    return x.double().pow(2).mean().sqrt().item()


def _long_cache(length, heads, dim, dev):
    """A cache of one request: random codes, scales and least values as rows of roughly normal values have them."""
    g = torch.Generator(dev).manual_seed(length)
    page = 64
    pages = -(-length // page)
    half = sa.Kv4Cache.padded_dim(dim) // 2
    u8 = lambda *s: torch.randint(0, 256, s, generator=g, device=dev, dtype=torch.uint8)  # noqa: E731

    def params():
        scale = 0.25 + 0.15 * torch.rand((pages, heads, page, 1), generator=g, device=dev)
        return torch.cat([scale, -7.5 * scale + 0.3 * torch.randn(scale.shape, generator=g, device=dev)], -1).to(BF16)

    return sa.Kv4Cache(u8(pages, heads, page, half), params(), u8(pages, heads, page // 4, half, 4), params(), dim)


def _attention64(cache, q, length):
    """q [H,D] over the whole cache: the result, and sum p (least + 8 scale), the mean that the codes' sums are added to."""
    per = q.shape[0] // cache.kv_heads
    qd = q.double().reshape(cache.kv_heads, per, -1) / math.sqrt(cache.dim)
    parts = [torch.arange(a, min(length, a + 65536), device=q.device, dtype=torch.int32) for a in range(0, length, 65536)]
    w = torch.softmax(torch.cat([torch.einsum("gpd,tgd->gpt", qd, cache.read(s)[0].double()) for s in parts], -1), -1)
    out = sum(torch.einsum("gpt,tgd->gpd", w[..., s[0]:s[-1] + 1], cache.read(s)[1].double()) for s in parts)
    page = cache.page_size
    par = torch.cat([cache.v_params[s.long() // page, :, s.long() % page].double() for s in parts])
    mean = torch.einsum("gpt,tg->gp", w, par[..., 1] + 8 * par[..., 0])
    return out.reshape(q.shape), mean


# requests that share the one cache, so that each request's blocks go to few warps
ATTEND = [(2000, 4, 64), (12000, 8, 64), (40000, 8, 64), (131072, 8, 64), (40000, 1, 2), (300000, 1, 2)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("spread", [0.02, 1.5], ids=["equal", "normal"])
@pytest.mark.parametrize("length,heads,requests", ATTEND)
def test_cache_attention_keeps_its_precision_over_long_caches(length, heads, requests, spread, dtype, dev):
    """Beside the output's own rounding the error is at most `own`, per unit of p:
    16 bits: a block's truncated sums (4 2^-23 of its parts) and sqrt(blocks of a
    warp) rounded additions (2^-24 each) of sums no larger than the parts, which
    are scale |code + offset|: 0.33 * 23.5 in bfloat16, 0.33 * 4 in float16.
    float32: the additions of the centred sums, which are as large as the result
    and the mean beside it; and 2^-20 for scores and probabilities of 24 bits."""
    cache = _long_cache(length, heads, 128, dev)
    q = (torch.randn(heads * 4, 128, generator=torch.Generator(dev).manual_seed(1), device=dev) * spread).to(dtype)
    tables = torch.arange(cache.num_pages, dtype=torch.int32, device=dev).expand(requests, -1).contiguous()
    lens = torch.full((requests,), length, dtype=torch.int32, device=dev)
    out = cache.attend(q.expand(requests, -1, -1), tables, lens)
    assert (out == out[:1]).all()
    ref, mean = _attention64(cache, q, length)
    adds = math.sqrt(length / 16 / 16)      # at least 16 warps to a request
    size, rounding = _rms(ref), _rms(ref.to(dtype).double() - ref)
    if dtype == F32:
        own = size * 2.0 ** -20 + adds * 2.0 ** -24 * (_rms(mean) + size)
    else:
        own = 0.33 * (23.5 if dtype == BF16 else 4.0) * (4 * 2.0 ** -23 + adds * 2.0 ** -24)
    err = _rms(out[0].double() - ref)
    assert err <= math.hypot(rounding, own) * 1.02, (err / size, rounding / size, own / size)


@pytest.mark.parametrize("dtype,d,dv", [(F32, 64, 64), (F32, 64, 128), (F32, 40, 32), (F16, 128, 128), (BF16, 128, 128), (BF16, 64, 80)])
@pytest.mark.parametrize("spread", [0.02, 1.5], ids=["equal", "normal"])
@pytest.mark.parametrize("n,m,window", [(512, 4608, 4096), (300, 700, 100), (2, 20000, None)], ids=["long", "short", "split"])
def test_windowed_attention_keeps_its_precision(n, m, window, spread, dtype, d, dv, dev):
    """float32: 24 truncated additions to a score (a sixth of a step each in the root
    mean square, of sums as large as the score, 3 in base 2) and 48 to a chain of two
    tiles of O: 2.7e-6 ln 2 and 1.4e-6 of the result.  16 bits: the probabilities'
    rounding, at most half a step of the type for all of a row alike, beside the output's own."""
    g = torch.Generator(dev).manual_seed(n + d)
    mk = lambda h, rows, w, s: (torch.randn(1, h, rows, w, generator=g, device=dev) * s).to(dtype)  # noqa: E731
    q, k, v = mk(4, n, d, spread), mk(2, m, d, 1.0), mk(2, m, dv, 1.0)
    out = sa.sliding_window_attention(q, k, v, window=window, sinks=5)
    kd, vd = (x[0].double().repeat_interleave(2, 0) for x in (k, v))
    sees = R.visible(n, m, window, 5).to(dev)
    x = torch.einsum("hnd,hmd->hnm", q[0].double(), kd) / math.sqrt(d)
    ref = torch.einsum("hnm,hmd->hnd", torch.softmax(x.masked_fill(~sees, -math.inf), -1), vd)
    size, rounding = _rms(ref), _rms(ref.to(dtype).double() - ref)
    own = size * (3.3e-6 if dtype == F32 else R.HALF[dtype])
    err = _rms(out[0].double() - ref)
    assert err <= math.hypot(rounding, own), (err / size, rounding / size, own / size)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("form,heads,m,dv,window", [("dense", 80, 131072, 64, None), ("dense", 80, 40000, 100, 30000), ("dense", 2, 300000, 64, None),
                                                   ("packed", 80, 60000, 64, None), ("packed", 3, 34000, 128, None)])
def test_windowed_attention_of_long_chains_is_not_low(form, heads, m, dv, window, dtype, dev):
    """Values of mean 1: the mean of the result beside that of the rounded reference
    (rounding has a mean of its own here: results crowd around 1, where the type's steps
    change).  The matrix units cut off 7e-8 for each 16 keys of a chain of at most 32768
    keys, 1.44e-4 in all.  A shift by that moves the rounded values of a share of
    1.44e-4 / step of the N elements by one step, so its mean is off by
    sqrt(1.44e-4 step / N) from it: four of those."""
    g = torch.Generator(dev).manual_seed(m)
    n, d = 256, 64
    q = torch.randn(1, heads, n, d, generator=g, device=dev).to(dtype)
    k, v = torch.empty(1, heads, m, d, dtype=dtype, device=dev), torch.empty(1, heads, m, dv, dtype=dtype, device=dev)
    for h in range(heads):
        k[0, h] = torch.randn(m, d, generator=g, device=dev).to(dtype)
        v[0, h] = (torch.randn(m, dv, generator=g, device=dev) + 1).to(dtype)
    if form == "dense":
        out = sa.sliding_window_attention(q, k, v, window=window)
    else:
        rows = lambda x: x[0].transpose(0, 1).contiguous()  # noqa: E731
        cu_q, cu_k = (torch.tensor([0, x], dtype=torch.int32, device=dev) for x in (n, m))
        out = sa.sliding_window_attention_packed(rows(q), rows(k), rows(v), cu_q, cu_k, window=window).transpose(0, 1)[None]
    at = torch.arange(m - n, m, device=dev)[:, None]
    j = torch.arange(m, device=dev)[None]
    for h in {0, heads - 1}:
        x = q[0, h].double() @ k[0, h].double().T / math.sqrt(d)
        x = torch.softmax(x.masked_fill((j > at) | (j <= at - (window or m)), -math.inf), -1)
        ref = x @ v[0, h].double()
        rounded = ref.to(dtype).double()
        low = 1 - (out[0, h].double().mean() / rounded.mean()).item()
        most = 2048 * 7e-8
        assert abs(low) <= most + 4 * math.sqrt(most * 2 * R.HALF[dtype] / ref.numel()), low
        err = _rms(out[0, h].double() - ref)
        assert err <= math.hypot(_rms(rounded - ref), _rms(ref) * R.HALF[dtype])
