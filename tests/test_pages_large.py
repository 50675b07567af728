"""Calls on the pages of large caches and batches: the kernels against the PyTorch forms (which
test_pages.py holds against walks over lists), and times that grow with the work and not its square."""

from __future__ import annotations

import pytest
import torch

from triton_flash_attention import paged_cache_compact

GPU = dict(device="cuda", dtype=torch.int32)


def microseconds(call, times=5):
    call()
    best = float("inf")
    for _ in range(times):
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        call()
        end.record()
        torch.cuda.synchronize()
        best = min(best, 1000 * begin.elapsed_time(end))
    return best


def cache(pages, free, B, M, seed=0):
    """A list that names ``free`` pages in any order, counts, and a table of any pages."""
    gen = torch.Generator("cuda").manual_seed(seed)
    names = torch.randperm(pages, generator=gen, device="cuda")[:free].int()
    shares = torch.randint(0, 5, (pages,), generator=gen, **GPU)
    shares[names.long()] = 0
    return torch.randint(-2, pages + 2, (B, M), generator=gen, **GPU), names, shares


@pytest.mark.gpu
@pytest.mark.parametrize(("pages", "free", "start"), [
    (1 << 19, 70000, None),
    ((1 << 19) + 1, 70000, 5),
    (300001, 150000, None),
    (700001, 700001, None),       # all of them
    (700001, 0, None),            # none
    (1 << 20, 1 << 19, 1000),     # whole chunks
    ((1 << 20) + 31, 40, None),
    (5000003, 4999000, 17),
    (5000003, 1300, -3),
])
def test_compact_kernel_of_many_pages(pages, free, start):
    table, names, shares = cache(pages, free, 37, 50, seed=pages % 1000)
    start = None if start is None else torch.tensor([start], **GPU)
    got = paged_cache_compact(table, names, shares, free_start=start, backend="triton")
    want = paged_cache_compact(table, names, shares, free_start=start, backend="torch")
    for name, a, b in zip(got._fields, got, want):
        assert torch.equal(a, b), name


@pytest.mark.gpu
def test_compact_kernel_where_a_page_is_named_twice():
    table, names, shares = cache(700000, 30000, 5, 50)
    names = torch.cat((names, names[:20000], torch.tensor([-1, 700000, 1 << 30], **GPU)))
    got = paged_cache_compact(table, names, shares, backend="triton")
    want = paged_cache_compact(table, names, shares, backend="torch")
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_compact_kernel_takes_no_time_that_grows_with_the_square():
    """Of 2^26 pages, within 100 times what copying the inputs takes (300 times where each
    of 2^16 blocks counts 2^21 words)."""
    table, names, shares = cache(1 << 26, 1 << 25, 256, 1024)
    out = [torch.empty_like(t) for t in (table, names, shares)]
    copies = microseconds(lambda: [a.copy_(b) for a, b in zip(out, (table, names, shares))])
    assert microseconds(lambda: paged_cache_compact(table, names, shares, backend="triton")) < 100 * copies
