"""Attention over a cache of more tokens than 2^30: window and first tokens past that.
One page holds the token that matters, another stands for all the rest."""

import math

import pytest
import torch

import serving_ref as R
import streaming_attention_b200 as sa
from test_kv4_gpu import _check_attend, _filled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window,sinks,at", [(None, 0, 0), (2 ** 30 + 500, 0, 512), (1, 2 ** 30 + 500, 2 ** 30)],
                         ids=["no-window", "window", "first-tokens"])
def test_windows_past_2_30_tokens(window, sinks, at):
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    dev, d, page, length = torch.device("cuda:0"), 32, 256, 2 ** 30 + 1000
    cache = sa.Kv4Cache.empty(2, 1, d, page_size=page, device=dev)
    ones = torch.ones(page, 1, d, device=dev)
    slots = torch.arange(2 * page, dtype=torch.int32, device=dev)
    cache.append(torch.cat([ones, 0 * ones]), torch.cat([3 * ones, -ones]), slots)
    tables = torch.ones(1, length // page + 1, dtype=torch.int32, device=dev)
    tables[0, at // page] = 0
    q = torch.full((1, 8, d), 4.0, dtype=torch.bfloat16, device=dev)
    out = cache.attend(q, tables, torch.tensor([length], dtype=torch.int32, device=dev), window=window, sinks=sinks)
    top = 4.0 * d / math.sqrt(d)
    others = (length if window is None else min(length, window + sinks)) - page
    w = others / (page * math.exp(top) + others)      # what the other tokens weigh
    # their sum, of 2^30 equal terms by 64 warps of eight lanes, is off by far less than a hundredth
    assert (out.double() - (3 - 4 * w)).abs().max() <= 2 ** -8 * 3 + 0.01 * 4 * w


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_many_first_tokens_and_a_short_window(dtype):
    """They count for how many CTAs share a request as a long window does."""
    dev, length = torch.device("cuda:0"), 9000
    cache, tables, lens, ks, vs = _filled(dev, [length], 2, 64, 64, torch.float32, 30)
    q = torch.randn(1, 2, 8, 64, generator=R.rng(31)).to(dtype).to(dev)
    for window, sinks in ((1, length), (64, 6000), (3, 4097)):
        _check_attend(cache.attend(q, tables, lens, window=window, sinks=sinks), q, ks, vs, [length], window, sinks)
