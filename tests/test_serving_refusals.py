"""Refusals of the serving entry points that look at tensors, on the CPU: no launch
is made."""

import pytest
import torch

import streaming_attention_b200 as sa
from streaming_attention_b200 import _serving


@pytest.fixture(autouse=True)
def no_launch(monkeypatch):
    monkeypatch.setattr(_serving, "device_of", lambda first, *others: first.device)
    monkeypatch.setattr(_serving, "launch", lambda *a: pytest.fail("launched"))


def test_results_are_not_written_to_expanded_tensors():
    x, cu = torch.zeros(6, 2, 64), torch.tensor([0, 6], dtype=torch.int32)
    for out in (torch.zeros(1, 2, 64).expand(6, -1, -1), torch.zeros(6, 1, 64).expand(-1, 2, -1)):
        with pytest.raises(ValueError, match="expanded"):
            sa.sliding_window_attention_packed(x, x, x, cu, cu, window=3, out=out)
        for pair in ((out, x), (x, out)):
            with pytest.raises(ValueError, match="expanded"):
                sa.qk_norm_rotary(x, x, torch.zeros(6, dtype=torch.int32), None, None, sa.rotary_frequencies(64), out=pair)


def test_release_takes_one_list_of_free_pages():
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match=r"free_pages must be \[F\]"):
        sa.release_kv_pages(i, i[:, None], torch.zeros(1, dtype=torch.bool), i[None], i, page_size=16)
