"""What long caches' calls may count on of the stream they are put on: all that stands
before them has ended when they start to read and to write."""

import glob
import os

import pytest
import torch

import streaming_attention_b200 as sa
from test_kv4_gpu import _filled
from test_long_cache_gpu import BF16, F32, _queries

CSRC = os.path.join(os.path.dirname(sa.__file__), "csrc")


def test_only_second_kernels_of_a_call_start_early():
    """A launch that may begin beside the kernel before it is sound where that kernel is the same call's: a prefix's
    sums and their join, scores and their weights.  An entry point's first kernel stands behind whatever the caller
    put on the stream."""
    early = {os.path.basename(p) for p in glob.glob(os.path.join(CSRC, "*.cu*"))
             if "ProgrammaticStreamSerialization" in open(p).read()}
    assert early == {"kv4_attend.cuh", "kv4_attend_weigh.cu"}
    # and there it is asked for in the one mode that always follows the prefix's kernel
    text = open(os.path.join(CSRC, "kv4_attend.cuh")).read()
    before, _ = text.split("attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization")
    assert before.rstrip().splitlines()[-1].strip().startswith("if (kMode == kTail) {")


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return torch.device("cuda:0")


@pytest.mark.gpu
@pytest.mark.parametrize("count", [4, 60])
def test_selection_sees_what_was_written_just_before(count, dev):
    """Queries, lengths, tables and bounds written by the launches before it, in every order of them."""
    cache, tables, lens, _, _ = _filled(dev, [700, 90, 333], 2, 64, 16, F32, 1)
    q = _queries(3, 1, 8, 64, BF16, 1, dev)
    bounds = cache.page_bounds()
    cache.update_page_bounds(bounds, tables, lens, lens)
    want = cache.select_pages(q, bounds, tables, lens, count=count)
    big = torch.empty(1 << 26, device=dev)
    q2, t2, l2 = torch.zeros_like(q), torch.zeros_like(tables), torch.ones_like(lens)
    for i in range(12):
        b2 = torch.zeros_like(bounds)
        q2.zero_(), t2.zero_(), l2.fill_(1)
        writes = [lambda: q2.copy_(q), lambda: t2.copy_(tables), lambda: l2.copy_(lens)]
        big.fill_(float(i))   # they wait for this one on the device, and the host runs ahead
        for k in range(2):
            writes[(i + k) % 3]()
        if i % 3 == 2:
            cache.update_page_bounds(b2, tables, lens, lens)
            writes[(i + 2) % 3]()
        else:
            writes[(i + 2) % 3]()
            cache.update_page_bounds(b2, t2, l2, l2)
        assert torch.equal(cache.select_pages(q2, b2, t2, l2, count=count), want)


@pytest.mark.gpu
def test_selection_in_memory_that_the_bounds_still_read(dev):
    """Copies of lengths and counts that the update made, and freed, are where the selection's output goes."""
    requests, h = 64, 1
    cache, tables, lens, _, _ = _filled(dev, [40 + r for r in range(requests)], h, 64, 16, F32, 2)
    q = _queries(requests, 1, 2, 64, BF16, 1, dev)
    want = cache.page_bounds()
    cache.update_page_bounds(want, tables, lens, lens)
    strided = torch.stack([lens, lens], -1)[:, 0]   # copied by the call
    big = torch.empty(1 << 26, device=dev)
    for i in range(20):
        bounds = cache.page_bounds()
        big.fill_(float(i))
        cache.update_page_bounds(bounds, tables, lens, strided)
        rows = [cache.select_pages(q, bounds, tables, lens, count=c, first=0, last=0) for c in (1, 1, 8, 8)]
        assert torch.equal(bounds, want)
        every = torch.arange(8, device=dev)
        pages = ((lens + 15) // 16)[:, None]
        for x in rows[2:]:
            assert torch.equal(x[:, 0, 0], torch.where(every < pages, every, -1).to(torch.int32))
