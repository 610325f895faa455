"""Float32 tensors that are contiguous but for the stride of an axis of one entry take
the tensor cores as their copies do: the same bits."""

import pytest
import torch

import serving_ref as R
import streaming_attention_b200 as sa

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return torch.device("cuda:0")


def _same(q, k, v, **kw):
    out = sa.sliding_window_attention(q, k, v, **kw)
    assert torch.equal(out, sa.sliding_window_attention(*(x.clone(memory_format=torch.contiguous_format) for x in (q, k, v)), **kw))
    per = q.shape[1] // k.shape[1]
    sees = R.visible(q.shape[2], k.shape[2], kw["window"], 0).to(q.device)
    for b in range(q.shape[0]):
        kd, vd = (x[b].double().repeat_interleave(per, 0) for x in (k, v))
        ref, spread, score = R.attention(q[b].double(), kd, vd, sees, 64 ** -0.5)
        R.assert_close(out[b], ref.cpu(), R.attention_bound(ref, spread, score, 64, k.shape[2], torch.float32, 0.0).cpu())


def test_one_key_head_of_tokens_first_tensors(dev):
    g = torch.Generator(dev).manual_seed(1)
    q = torch.randn(2, 4, 700, 64, generator=g, device=dev)
    k, v = (torch.randn(2, 700, 1, 64, generator=g, device=dev).transpose(1, 2) for _ in range(2))
    assert k.is_contiguous() and k.stride(1) == 64
    _same(q, k, v, window=300)


def test_one_token_of_tokens_first_tensors(dev):
    g = torch.Generator(dev).manual_seed(2)
    q = torch.randn(2, 1, 4, 64, generator=g, device=dev).transpose(1, 2)
    k, v = (torch.randn(2, 2, 900, 64, generator=g, device=dev) for _ in range(2))
    assert q.is_contiguous() and q.stride(2) != 64
    _same(q, k, v, window=None)


def test_the_front_of_a_longer_buffer(dev):
    g = torch.Generator(dev).manual_seed(3)
    q = torch.randn(1, 1, 500, 64, generator=g, device=dev)
    k, v = (torch.randn(1, 1, 4000, 64, generator=g, device=dev)[:, :, :600] for _ in range(2))
    assert k.is_contiguous() and k.stride(1) == 4000 * 64
    _same(q, k, v, window=400)
