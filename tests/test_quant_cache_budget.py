"""How much of the free memory becomes pages, without a GPU: what prompt portions read back of an 8-bit cache stays free."""
import pytest
import torch

from ginfer_b200.cache.storage import plan_groups
from ginfer_b200.engine.runner import ModelRunner
from ginfer_b200.ops import quant_cache as qc
from ginfer_b200.parts.base import PagedKVSpec


def runner(specs, eager=True, seqs=64, longest=131072, tokens=8192, page=16):
    r = object.__new__(ModelRunner)
    r.groups, _ = plan_groups(specs)
    r.device, r.page_size, r.max_num_seqs, r.max_seq_len = "cuda:0", page, seqs, longest
    r.max_num_batched_tokens, r.enforce_eager = tokens, eager
    return r


def taken(r, counts, itemsize):
    return sum(n * g.bytes_per_page(r.page_size, itemsize) for n, g in zip(counts, r.groups))


@pytest.mark.parametrize("itemsize", [2, 4])
@pytest.mark.parametrize("eager", [True, False])
@pytest.mark.parametrize("window", [0, 4096])
def test_the_read_back_fits_beside_the_pages(monkeypatch, itemsize, eager, window):
    free = 40 << 30
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device=None: (free, 180 << 30))
    r = runner({i: PagedKVSpec(8, 128, window, kept="int8") for i in range(32)}, eager, seqs=10 ** 6)
    counts = r._page_counts(None, 1.0, itemsize)
    # one request of 131,072 tokens, or a window and a portion of it, a layer at a time
    seen = 131072 if not window else max(qc.READ_AT_ONCE, 4096 + 8192)
    dense = 2 * seen * 8 * 128 * itemsize * (1 if eager else 2)
    left = free - taken(r, counts, itemsize)
    page = r.groups[0].bytes_per_page(16, itemsize)
    assert dense <= left < dense + page
    assert r._page_counts(None, 0.5, itemsize)[0] == pytest.approx(counts[0] / 2, abs=1)


def test_other_caches_get_what_they_got(monkeypatch):
    free = 40 << 30
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device=None: (free, 180 << 30))
    r = runner({i: PagedKVSpec(8, 128) for i in range(32)}, seqs=10 ** 6)
    assert r._page_counts(None, 0.8, 2) == [int(free * 0.8) // r.groups[0].bytes_per_page(16, 2)]
    # a count that is asked for is kept
    r = runner({0: PagedKVSpec(8, 128, kept="fp8")})
    assert r._page_counts(100, 0.8, 2) == [100]
    # and there is a page, however little is free
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device=None: (1 << 20, 180 << 30))
    assert r._page_counts(None, 0.8, 2) == [1]


@pytest.mark.parametrize("page,window", [(16, 0), (16, 100), (7, 100), (16, 5000), (24, 200000)])
def test_bytes_hold_every_group_of_portions(page, window):
    """No group of portions that a step makes takes more."""
    longest, portion = 40000, 2048
    most = qc.read_back_bytes(2, 64, 2, page, longest, portion, window)
    W = -(-longest // page)
    for starts, counts in (([0], [portion]), ([longest - portion], [portion]), ([30000, 0, 5], [1000, 500, 548]),
                           ([100] * 40, [50] * 40), ([longest - 64] * 32, [64] * 32)):
        for capturing in (False, True):
            pages = qc.portion_pages(starts, counts, page, window, W, capturing)
            for i, j in qc.portion_groups(pages, page):
                assert 2 * (j - i) * max(pages[i:j]) * page * 2 * 64 * 2 <= most
