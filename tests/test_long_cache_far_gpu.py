"""A shared prefix that ends where 31 bits do."""

import math

import pytest
import torch

import long_cache_ref as L
import serving_ref as R
import streaming_attention_b200 as sa
from test_long_cache_gpu import BF16, F16, P_SHARED, _close, _i32, _queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requests", [3, 40])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_prefix_up_to_the_last_position(requests, dtype):
    """Pages of 16, whose table reaches 2^31 - 16: the last tile of 64 tokens ends behind it, and the prefix within it."""
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    dev, d, page, own, window = torch.device("cuda:0"), 64, 16, 3, 100
    width = (2 ** 31 - 16) // page
    prefix = width * page - 6
    cache = sa.Kv4Cache.empty(9 + requests, 1, d, page_size=page, device=dev)
    g = R.rng(1)
    rows = cache.num_pages * page
    slots = torch.arange(rows, dtype=torch.int32, device=dev)
    cache.append(torch.randn(rows, 1, d, generator=g).to(dev), (torch.randn(rows, 1, d, generator=g) + 2).to(dev), slots)
    k, v = (x.cpu().double() for x in cache.read(slots))
    table = torch.zeros(width, dtype=torch.int32, device=dev)
    table[-9:] = torch.arange(9, dtype=torch.int32, device=dev)
    tables = 9 + torch.arange(requests, dtype=torch.int32, device=dev)[:, None]
    q = _queries(requests, 1, 2, d, dtype, 2, dev)
    out = cache.attend_shared(q, table, _i32([prefix], dev), tables, _i32([own] * requests, dev), window=window)
    for r in range(requests):
        # the last 9 * 16 - 6 tokens of the prefix and the own ones, of which the window leaves 100
        at = list(range(9 * page - 6)) + [(9 + r) * page + i for i in range(own)]
        sees = R.visible(1, len(at), window, 0)
        ref, spread, score, _ = L.attend(q[r].cpu().double(), k[at], v[at], sees, 1 / math.sqrt(d))
        _close(out[r], ref, spread, score, d, len(at), P_SHARED[dtype])
    sa.check_serving_status(dev)
