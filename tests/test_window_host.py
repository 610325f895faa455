"""Which 16-bit windowed calls are given a workspace for split keys, on the CPU: the
library's rule alone decides."""

import ctypes

import pytest
import torch

import streaming_attention_b200 as sa
from streaming_attention_b200 import _lib, window

CASES = [
    # b, h, hkv, n, m, d, window, split
    (1, 32, 8, 1, 4096, 128, None, True), (1, 32, 8, 128, 4096, 128, None, True), (1, 32, 8, 256, 4096, 128, None, True),
    (1, 32, 8, 512, 4096, 128, None, False), (1, 32, 8, 512, 8192, 128, None, True), (1, 8, 8, 1024, 32768, 64, None, True),
    (1, 32, 8, 600, 16000, 128, None, False), (1, 32, 8, 1, 3008, 128, None, False), (1, 32, 8, 1, 8192, 128, 1024, False),
    (16, 32, 8, 1, 4096, 128, None, False), (1, 8, 8, 2304, 8192, 128, None, True),
]


@pytest.mark.parametrize("case", CASES, ids=["-".join(map(str, c)) for c in CASES])
def test_the_librarys_rule_decides(case, monkeypatch):
    b, h, hkv, n, m, d, win, split = case
    got = []
    monkeypatch.setattr(window.S, "device_of", lambda first, *others: first.device)
    monkeypatch.setattr(window.S, "launch", lambda dev, name, *args: got.append(args))
    q, k = torch.empty(b, h, n, d, dtype=torch.bfloat16), torch.empty(b, hkv, m, d, dtype=torch.bfloat16)
    sa.sliding_window_attention(q, k, k, window=win)
    size = ctypes.c_size_t(0)
    _lib.check(_lib.load().sa_window_attention_workspace_size(b, h, hkv, n, m, d, d, win or 0, 0, _lib.REP_DTYPES["bfloat16"],
                                                              ctypes.byref(size)), "size")
    assert (size.value > 0) == split
    assert got[0][-1] == size.value and (got[0][-2] is not None) == split
