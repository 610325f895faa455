"""How precise the attention behind a shared prefix stays as the prefix grows: an error
that grows with its length, and that the bounds for single elements, which grow too, let pass."""

import math

import pytest
import torch

import serving_ref as R
import streaming_attention_b200 as sa

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _rms(x):
    return x.double().pow(2).mean().sqrt().item()


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("spread", [0.02, 1.5], ids=["equal", "normal"])
@pytest.mark.parametrize("prefix,requests,n,heads,h,window", [
    (40000, 100, 3, 64, 8, None), (131072, 100, 3, 64, 8, None), (300000, 100, 3, 64, 8, None),
    (200000, 100, 3, 64, 8, 100000), (131072, 40, 1, 8, 1, None)])
def test_shared_prefix_of_long_chains_is_not_low(prefix, requests, n, heads, h, window, spread, dtype):
    """Many rows, so that few CTAs share the prefix, and values of mean 1: the mean of the result beside that of the
    rounded reference.  The matrix units cut off 7e-8 for each 16 tokens of a chain of at most 32768, 1.44e-4 in all;
    a shift by that moves the rounded values of a share of 1.44e-4 / step of the N elements by one step, so its mean
    is off by sqrt(1.44e-4 step / N) from it: four of those.  The error as a whole: the result's rounding, that shift, and
    the float16 roundings of probabilities and values, half a step (2^-11) of each term from either."""
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    dev, d, page, own = torch.device("cuda:0"), 64, 64, 3
    g = torch.Generator(dev).manual_seed(prefix)
    pages = -(-prefix // page)
    cache = sa.Kv4Cache.empty(pages + requests, h, d, page_size=page, device=dev)
    for a in range(0, prefix, 65536):
        s = torch.arange(a, min(prefix, a + 65536), dtype=torch.int32, device=dev)
        cache.append(torch.randn(len(s), h, d, generator=g, device=dev), torch.randn(len(s), h, d, generator=g, device=dev) + 1, s)
    tables = pages + torch.arange(requests, dtype=torch.int32, device=dev)[:, None]
    s = (tables * page + torch.arange(own, dtype=torch.int32, device=dev)).flatten()
    cache.append(torch.randn(len(s), h, d, generator=g, device=dev), torch.randn(len(s), h, d, generator=g, device=dev) + 1, s)
    q = (torch.randn(requests, n, heads, d, generator=g, device=dev) * spread).to(dtype)
    out = cache.attend_shared(q, torch.arange(pages, dtype=torch.int32, device=dev),
                              torch.tensor([prefix], dtype=torch.int32, device=dev), tables,
                              torch.full((requests,), own, dtype=torch.int32, device=dev), window=window)
    m, got, want = prefix + own, [], []
    j = torch.arange(m, device=dev)
    for r in {0, 7, requests - 1}:
        slots = torch.cat([torch.arange(prefix, dtype=torch.int32, device=dev), s[r * own:(r + 1) * own]])
        k, v = cache.read(slots)
        at = torch.arange(m - n, m, device=dev)[:, None]
        hidden = (j > at) | (j <= at - (window or m))
        for x in range(h):
            mine = slice(x * (heads // h), (x + 1) * (heads // h))
            p = torch.einsum("npd,td->pnt", q[r, :, mine].double(), k[:, x].double()) / math.sqrt(d)
            p = torch.softmax(p.masked_fill_(hidden, -math.inf), -1)
            want.append((p @ v[:, x].double()).transpose(0, 1).flatten())
            got.append(out[r, :, mine].double().flatten())
    got, ref = torch.cat(got), torch.cat(want)
    rounded = ref.to(dtype).double()
    low, most = 1 - (got.mean() / rounded.mean()).item(), 2048 * 7e-8
    assert abs(low) <= most + 4 * math.sqrt(most * 2 * R.HALF[dtype] / ref.numel()), low
    own_error = _rms(ref) * (2 * 2.0 ** -11 + most)
    assert _rms(got - ref) <= math.hypot(_rms(rounded - ref), own_error)
