"""Calls on the pages of large caches and batches: the kernels against the PyTorch forms (which
test_pages.py holds against walks over lists), and times that grow with the work and not its square."""

from __future__ import annotations

import pytest
import torch
from test_prefix_work import Workspaces

from triton_flash_attention import paged_cache_compact, paged_cache_fork

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


def rows(B, M, pages, parents, seed=0):
    """Rows of any pages of which several may be the same, with counts that cover them."""
    gen = torch.Generator("cuda").manual_seed(seed)
    table = torch.randint(-1, pages, (B, M), generator=gen, **GPU)
    lengths = torch.randint(0, 16 * M + 9, (B,), generator=gen, **GPU)
    par = torch.randint(-1, B, (B,), generator=gen, **GPU)
    if isinstance(parents, int):
        par[:] = parents
    elif parents is not None:  # neighbours with one parent, which one of them may be itself
        n, which = parents
        par = (torch.arange(B, **GPU) // n * n + which).clamp(max=B - 1)
    shares = torch.randint(0, 40, (pages,), generator=gen, **GPU)
    names = torch.randperm(pages, generator=gen, device="cuda").int()
    return table, lengths, par, names, shares


@pytest.mark.gpu
@pytest.mark.parametrize("pages", [8000, 70000])
@pytest.mark.parametrize(("B", "M", "parents"), [
    (4096, 3, None), (4097, 3, None), (4097, 1500, 9), (30001, 2, None), (131071, 1, None), (131071, 2, 70000),
    (20000, 2, -1), (5000, 2, (8, 0)), (5000, 2, (100, 37)), (5001, 2, (200, 150)), (5001, 2, (64, 64)),
])
def test_fork_kernel_of_many_rows(B, M, parents, pages):
    outs = []
    for backend in ("triton", "torch"):
        table, lengths, par, names, shares = rows(B, M, pages, parents, seed=B + M)
        fork = paged_cache_fork(table, lengths, par, names, shares, page_size=16,
                                free_start=torch.tensor([pages // 2], **GPU), backend=backend)
        outs.append(dict(fork._asdict(), table=table, names=names, shares=shares))
    for name in outs[0]:
        assert torch.equal(outs[0][name], outs[1][name]), name


@pytest.mark.gpu
def test_fork_kernel_takes_no_time_that_grows_with_the_square():
    """16 times the rows in less than 32 times the time (78 times where each row looks through all
    parents)."""
    times = []
    for B in (8191, 131071):
        table, lengths, par, names, shares = rows(B, 1, 8000, None)
        shares += 1 << 20
        times.append(microseconds(lambda: paged_cache_fork(
            table, lengths, par, names, shares, page_size=16, backend="triton")))
    assert times[1] < 32 * times[0]


@pytest.mark.gpu
@pytest.mark.parametrize(("B", "pages"), [
    (9, 500), (900, 8192), (1500, 8000), (1500, 8193), (37, 100001), (5000, 4000), (5000, 50000),
])
def test_pages_kernels_stay_inside_their_workspaces(B, pages, monkeypatch):
    """Workspaces of exactly the bytes that the calls ask for, between guards."""
    kept = Workspaces(monkeypatch)
    table, lengths, par, names, shares = rows(B, 5, pages, None)
    state = [t.clone() for t in (table, names, shares)]
    got = paged_cache_fork(state[0], lengths, par, state[1], state[2], page_size=16, backend="triton")
    kept.last()
    want = paged_cache_fork(table, lengths, par, names, shares, page_size=16, backend="torch")
    assert all(torch.equal(a, b) for a, b in zip((*got, *state), (*want, table, names, shares)))


@pytest.mark.gpu
@pytest.mark.parametrize(("B", "pages"), [(9, 500), (9, 14001), (900, 16000), (37, 100001), (5, 600001)])
def test_compact_kernels_stay_inside_their_workspaces(B, pages, monkeypatch):
    kept = Workspaces(monkeypatch)
    table, names, shares = cache(pages, pages // 3, B, 5)
    got = paged_cache_compact(table, names, shares, backend="triton")
    kept.last()
    want = paged_cache_compact(table, names, shares, backend="torch")
    assert all(torch.equal(a, b) for a, b in zip(got, want))
