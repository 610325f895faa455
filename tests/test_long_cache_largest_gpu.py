"""A shared prefix with rows so large that the row's last code would pass float32, though
what the row holds does not."""

import math

import pytest
import torch

import long_cache_ref as L
import serving_ref as R
import streaming_attention_b200 as sa
from test_long_cache_gpu import BF16, P_SHARED, _close, _i32, _queries

pytestmark = pytest.mark.gpu


# (keys: by the tensor cores' kernel.  The others, as `attend`, take codes plus 16 and scales apart, so they hold keys of
# 2^128 / 31 steps at most.)
@pytest.mark.parametrize("every", [False, True], ids=["one", "all"])
@pytest.mark.parametrize("which,requests", [("k", 40), ("v", 2), ("v", 40)])
def test_rows_at_the_end_of_float32(requests, which, every):
    """Own lengths of 3 and 83 behind 640 tokens and a window of 200: the first kind sees tokens 443.., the other 523..  The token
    of 1.9 2^127 (a value) or 2^124 (a key, with queries of 2^-126) is the 460th: or every one of the prefix is so large.
    Who sees none of them must not notice."""
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    dev, d, page, prefix, window = torch.device("cuda:0"), 64, 64, 640, 200
    g = R.rng(2)
    lengths = [3 + 80 * (r % 2) for r in range(requests)]
    cache = sa.Kv4Cache.empty(10 + 2 * requests, 1, d, page_size=page, device=dev)
    rows = cache.num_pages * page
    slots = torch.arange(rows, dtype=torch.int32, device=dev)
    cache.append(torch.randn(rows, 1, d, generator=g).to(dev), torch.randn(rows, 1, d, generator=g).to(dev), slots)
    for at in range(prefix) if every else [460]:
        p, o = at // page, at % page
        if which == "v":   # codes 0 and 1: 1.9 2^127 and 2^121 more; 15 times that would pass 2^128
            cache.v_codes[p, 0, o // 4, :, o % 4] = 0x10
            cache.v_params[p, 0, o] = torch.tensor([2.0 ** 121, 1.8984375 * 2.0 ** 127]).to(BF16)
        else:   # codes 0 and 1: -2^124 and 2^124; 8 times the scale would pass 2^128
            cache.k_codes[p, 0, o] = torch.randint(0, 2, (d // 2,), generator=g).to(torch.uint8).to(dev) * 16 + (at & 1)
            cache.k_params[p, 0, o] = torch.tensor([2.0 ** 125, -(2.0 ** 124)]).to(BF16)
    k, v = (x.cpu().double() for x in cache.read(slots))
    assert torch.isfinite(k).all() and torch.isfinite(v).all()
    tables = 10 + 2 * torch.arange(requests, dtype=torch.int32)[:, None] + torch.tensor([0, 1], dtype=torch.int32)
    q = _queries(requests, 1, 2, d, BF16, 3, dev) * (2.0 ** -126 if which == "k" else 1)
    out = cache.attend_shared(q, torch.arange(10, dtype=torch.int32, device=dev), _i32([prefix], dev), tables.to(dev),
                              _i32(lengths, dev), window=window)
    for r, x in enumerate(lengths):
        at = list(range(prefix)) + [int(tables[r, j // page]) * page + j % page for j in range(x)]
        sees = R.visible(1, prefix + x, window, 0)
        ref, spread, score, _ = L.attend(q[r].cpu().double(), k[at], v[at], sees, 1 / math.sqrt(d))
        _close(out[r], ref, spread, score, d, prefix + x, P_SHARED[BF16])
