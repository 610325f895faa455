"""Windowed attention where a value that is not finite stands in a tile, seen or
hidden, and where the scale is zero."""

import os

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
