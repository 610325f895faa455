"""The persistent 16-bit window kernel over many query tile pairs, with gaps
between the first tokens' key tiles and the windows': what hands scores,
probabilities and products from warp to warp, at each change of pair and across
each gap.  Every element is held against the float64 masked softmax."""

import pytest
import torch

import serving_ref as R
import streaming_attention_b200 as sa

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return torch.device("cuda:0")


def _check(q, k, v, out, window, sinks):
    """One [H,N,D] sequence at a time, on the GPU."""
    sees = R.visible(q.shape[2], k.shape[2], window, sinks).to(q.device)
    per = q.shape[1] // k.shape[1]
    keys = min(k.shape[2], (window or k.shape[2]) + sinks)
    for b in range(q.shape[0]):
        kd, vd = (x[b].double().repeat_interleave(per, 0) for x in (k, v))
        ref, spread, score = R.attention(q[b].double(), kd, vd, sees, q.shape[-1] ** -0.5)
        bound = R.attention_bound(ref, spread, score, q.shape[-1], keys, out.dtype, R.HALF[out.dtype])
        R.assert_close(out[b], ref.cpu(), bound.cpu())


# ungrouped heads: a query tile is 128 queries, and a window that is small against
# it leaves tiles between first tokens and window that nobody in the tile needs
@pytest.mark.parametrize("d", [16, 128])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("n,m,window,sinks", [(300, 300, 20, 49), (300, 300, 5, 64), (513, 600, 1, 64), (400, 400, 70, 128),
                                             (260, 900, 130, 57), (385, 385, 1, 128), (257, 257, 40, 0)])
def test_gaps_between_first_tokens_and_windows(n, m, window, sinks, dtype, d, dev):
    g = torch.Generator(dev).manual_seed(n + sinks)
    mk = lambda rows, s: (torch.randn(6, 40, rows, d, generator=g, device=dev) * s).to(dtype)  # noqa: E731
    q, k, v = mk(n, 1.5), mk(m, 1.0), mk(m, 1.0)
    out = sa.sliding_window_attention(q, k, v, window=window, sinks=sinks)
    _check(q, k, v, out, window, sinks)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_many_short_pairs(dtype, dev):
    """Thousands of pairs of one to three key tiles each: nearly all the time is pair changes; the same bits each time."""
    g = torch.Generator(dev).manual_seed(3)
    q, k, v = ((torch.randn(64, 32, 130, 64, generator=g, device=dev)).to(dtype) for _ in range(3))
    first = sa.sliding_window_attention(q, k, v, window=30, sinks=2)
    _check(q[:4], k[:4], v[:4], first[:4], 30, 2)
    for _ in range(5):
        assert torch.equal(first, sa.sliding_window_attention(q, k, v, window=30, sinks=2))


def test_many_short_packed_pairs(dev):
    """A ragged batch of hundreds of requests, some empty, over the whole chip."""
    g = torch.Generator(dev).manual_seed(4)
    n = torch.randint(0, 140, (700,), generator=torch.Generator().manual_seed(5)).tolist()
    t = sum(n)
    q, k, v = ((torch.randn(t, h, 64, generator=g, device=dev)).to(BF16) for h in (4, 4, 4))
    cu = torch.tensor([0] + n, device=dev).cumsum(0).to(torch.int32)
    out = sa.sliding_window_attention_packed(q, k, v, cu, cu, window=20, sinks=49)
    at = 0
    for x in n[:200]:
        rows = slice(at, at + x)
        if x:
            _check(*(y[None, rows].transpose(1, 2) for y in (q, k, v, out)), 20, 49)
        at += x


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("h,hkv,n,m,d,window,sinks", [(32, 8, 256, 4096, 128, None, 0), (8, 8, 520, 5000, 64, 4500, 3),
                                                     (32, 8, 512, 9000, 64, None, 0), (4, 2, 1030, 12000, 80, 11000, 70)])
def test_hundreds_of_queries_over_split_keys(h, hkv, n, m, d, window, sinks, dtype, dev):
    """Too few pairs for the chip though the rows are many: their keys are split, and joined."""
    g = torch.Generator(dev).manual_seed(n)
    q, k, v = (torch.randn(1, x, y, d, generator=g, device=dev).to(dtype) for x, y in ((h, n), (hkv, m), (hkv, m)))
    out = sa.sliding_window_attention(q, k, v, window=window, sinks=sinks)
    for x in range(0, h, h // 2):
        y = x // (h // hkv)
        _check(q[:, x:x + 1], k[:, y:y + 1], v[:, y:y + 1], out[:, x:x + 1], window, sinks)
    assert torch.equal(out, sa.sliding_window_attention(q, k, v, window=window, sinks=sinks))
