"""Pages that sequences share in the paged key/value cache (csrc/fa_pages.hip): rows of the page
table that fork, change places and end, the pages' copies, and the compaction of the cache.

Beside what :mod:`.paged` keeps, a program keeps ``page_shares`` [pages] (int32): how many hold a
page beyond its first holder, so 0 for a page that :func:`.paged.paged_cache_plan` hands out, and
``free_pages`` as a stack: the pages from ``free_start`` on are free, the plan takes the first of
them, and pages that are given up go back in front of them. A list with room for all pages never
overflows. Everything stays on the GPU, and no kernel's call reads it on the host.

A step of beam search, where row b of the next step continues row ``parents[b]``:

    fork = paged_cache_fork(table, lengths, parents, free_pages, page_shares, page_size=16,
                            free_start=free_start)
    for key_cache, value_cache in layers:
        paged_cache_copy(key_cache, value_cache, fork.sources, fork.targets, tokens=fork.tokens)
    lengths, free_start = fork.lengths, fork.free_start

Samples of one prompt are rows with the same parent; a sequence ends where its row's parent is -1.
A begun page, the last of a sequence that does not fill it, has to be held by one row alone, as it is
after forks and plans: a program that shortens a row into a shared page copies this page first.
The rows of a fork share whole pages, which :func:`.prefix.paged_prefix_attention` reads once.

No counterpart in the reference. Names, checks and the choice of a backend follow :mod:`.paged`.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _ops
from .attention import Backend, _forward_ad_active
from .paged import _PAGE_MULTIPLE, _cache_reason, _check_caches, _check_ints, _check_table
from .rotary import _binding, _check_backend, _check_tensor, _falls_back, _gpu_reason

_MOST = 1 << 30  # pages, entries of a list


class PagedFork(NamedTuple):
    """The new rows' lengths and the copies that they need (:func:`paged_cache_fork`)."""

    lengths: torch.Tensor     # [B] int32
    sources: torch.Tensor     # [B] int32, the page that row b's begun page is copied from, or -1
    targets: torch.Tensor     # [B] int32, the page that it is copied to, or -1
    tokens: torch.Tensor      # [B] int32, the tokens that it holds
    free_start: torch.Tensor  # [1] int32, place of the first free page


class PagedCompaction(NamedTuple):
    """A compacted cache's bookkeeping and its moves (:func:`paged_cache_compact`)."""

    page_table: torch.Tensor   # [B, M] int32
    free_pages: torch.Tensor   # [F] int32
    page_shares: torch.Tensor  # [pages] int32
    sources: torch.Tensor      # [F] int32, the pages that move, -1 behind the last
    targets: torch.Tensor      # [F] int32, where they move to
    used: torch.Tensor         # [1] int32, pages that are held: 0 .. used - 1


def _check_start(free_start, device) -> None:
    if free_start is None:
        return
    _check_tensor("free_start", free_start, free_start.ndim if isinstance(
        free_start, torch.Tensor) else 1, "(1,)")
    if free_start.numel() != 1 or free_start.dtype != torch.int32 or free_start.device != device:
        raise ValueError(f"free_start must be one int32 value on {device}")


def _check_lists(page_table, free_pages, page_shares, free_start) -> None:
    device = page_table.device
    for name, t, shape in (("free_pages", free_pages, "(free pages,)"),
                           ("page_shares", page_shares, "(pages,)")):
        _check_tensor(name, t, 1, shape)
        _check_ints(name, t, tuple(t.shape), device)
    if page_shares.shape[0] == 0:
        raise ValueError("page_shares must have at least one page")
    _check_start(free_start, device)


def _start(free_start, free_pages):
    zero = torch.zeros(1, dtype=torch.int64, device=free_pages.device)
    return zero if free_start is None else free_start.reshape(1).long().clamp(0, free_pages.shape[0])


# ---- fork -------------------------------------------------------------------------------


def _torch_fork(page_table, lengths, parents, free_pages, page_shares, free_start, page_size):
    S, (B, M), P, F = page_size, page_table.shape, page_shares.shape[0], free_pages.shape[0]
    device = page_table.device
    start = _start(free_start, free_pages)
    old, length = page_table.clone(), lengths.long().clamp(min=0)
    held = (length + S - 1) // S
    begun = torch.where(held <= M, length % S, 0)
    held = held.clamp(max=M)
    rows, j = torch.arange(B, device=device), torch.arange(M, device=device)
    live = (parents >= 0) & (parents < B)
    par = torch.where(live, parents, 0).long()
    known = (old >= 0) & (old < P)
    if B:
        children = torch.zeros(B, dtype=torch.int64, device=device).index_add_(0, par, live.long())
        # the child that goes on in the begun page: the row itself, or its first child
        rank = torch.where(live, torch.where(par == rows, -1, rows), B)
        keeper = torch.full((B,), B, dtype=torch.int64, device=device)
        keeper = keeper.scatter_reduce(0, par, rank, "amin")
        last = (j == held[:, None] - 1) & (begun > 0)[:, None]
        change = torch.where(last, children.clamp(max=1)[:, None], children[:, None]) - 1
        change = torch.where((j < held[:, None]) & known, change, 0)
        page_shares.index_add_(0, torch.where(known, old, 0).flatten().long(),
                               change.flatten().to(torch.int32))
        end = (held[par] - 1).clamp(min=0)
        source = old[par, end]
        copies = live & (begun[par] > 0) & (rank != keeper[par]) & known[par, end]
    else:
        source, copies = parents, live
    place = start + torch.cumsum(copies.long(), 0) - 1
    targets = torch.full((B,), -1, dtype=torch.int32, device=device)
    if F:
        targets = torch.where(copies & (place < F), free_pages[place.clamp(0, F - 1)], targets)
    if B:
        new = torch.where((j < held[par][:, None]) & live[:, None], old[par], old)
        page_table.copy_(torch.where(copies[:, None] & (j == end[:, None]), targets[:, None], new))
    # the pages that nobody holds go in front of the free ones that are left
    gone = page_shares < 0
    page_shares.clamp_(min=0)
    first = start + torch.minimum(copies.sum(), F - start) - gone.sum()
    released = torch.nonzero(gone).squeeze(1)
    at = first + torch.arange(released.shape[0], device=device)
    free_pages[at[at >= 0]] = released[at >= 0].to(torch.int32)
    return PagedFork(torch.where(live, length[par] if B else length, 0).to(torch.int32),
                     torch.where(copies, source, -1).to(torch.int32), targets,
                     torch.where(copies, begun[par] if B else begun, 0).to(torch.int32),
                     first.clamp(min=0).to(torch.int32))


def paged_cache_fork(
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    parents: torch.Tensor,
    free_pages: torch.Tensor,
    page_shares: torch.Tensor,
    *,
    page_size: int,
    free_start: torch.Tensor | None = None,
    backend: Backend = "auto",
) -> PagedFork:
    """Row b of the page table becomes the old row ``parents[b]``, sharing its pages, or is given
    up where that is no row (-1).

    ``page_table`` [B, M], ``free_pages`` [F] and ``page_shares`` [pages] are changed in place
    (all integers are int32): a new row's entries for the tokens it holds are written, no others.
    A row's whole pages are shared by all its children. Its begun page, the last one where its
    tokens do not fill it, goes on with one of them, the row itself if it is its own child, else
    the first; each other child b takes the first free page that is left, ``targets[b]``, into
    which :func:`paged_cache_copy` has to copy the first ``tokens[b]`` rows of page ``sources[b]``
    in every layer's caches (-1, -1 and 0 where nothing is to be copied). Pages that nobody holds
    any more return to the list, in ascending order in front of the free ones that are left.

    Where the free pages do not suffice, ``targets`` and the entries of the missing ones are -1,
    with their ``sources`` named. Negative lengths are taken as 0, ``free_start`` into [0, F].
    Entries that name no page hold none and are handed on as they are. ``page_shares`` has to count
    the holders: where it does not, pages may return too early or never.
    """
    native = _binding(backend)
    if native is not None:
        out = native.paged_fork(page_table, lengths, parents, free_pages, page_shares, page_size,
                                free_start)
        if out is not None:
            return PagedFork(*out)
    _check_backend(backend)
    _check_table(page_table, page_size)
    B, device = page_table.shape[0], page_table.device
    for name, t in (("lengths", lengths), ("parents", parents)):
        _check_ints(name, t, (B,), device)
    _check_lists(page_table, free_pages, page_shares, free_start)
    if B > 1 and page_table.stride(0) < page_table.shape[1]:
        raise ValueError("the rows of page_table must not overlap")
    for name, t in (("free_pages", free_pages), ("page_shares", page_shares)):
        if t.shape[0] > 1 and t.stride(0) == 0:
            raise ValueError(f"{name} must not be an expanded tensor")
    reason = None
    if backend != "torch":
        reason = _gpu_reason(page_table)
        if reason is None and page_table.stride(1) != 1 and page_table.shape[1] > 1:
            reason = "the rows of page_table must be contiguous"
        elif reason is None and not (free_pages.is_contiguous() and page_shares.is_contiguous()):
            reason = "free_pages and page_shares must be contiguous"
        elif reason is None and (B >= 1 << 17 or max(free_pages.shape[0], page_shares.shape[0]) >= _MOST):
            reason = "too many sequences or pages for one launch"
    if _falls_back(backend, reason):
        return _torch_fork(page_table, lengths, parents, free_pages, page_shares, free_start,
                           page_size)
    return PagedFork(*_ops.paged_fork(page_table, lengths, parents, free_pages, page_shares,
                                      free_start, page_size))


# ---- copy -------------------------------------------------------------------------------


def paged_cache_copy(
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    sources: torch.Tensor,
    targets: torch.Tensor,
    *,
    tokens: torch.Tensor | None = None,
    backend: Backend = "auto",
) -> None:
    """Copy pages of the caches [pages, Hkv, page_size, D] into others, in place.

    Page ``sources[i]`` goes to page ``targets[i]`` ([n], int32), all of it or its first
    ``tokens[i]`` rows (int32, taken into [0, page_size]); the target's other rows stay as they
    were. Pairs of which one names no page (-1) are left out. The targets must differ from each
    other and from all sources. Gradients are not recorded: the call raises where one would have
    to be. Tangents move along: inside a forward-mode level the call runs in PyTorch under
    ``backend="auto"``.
    """
    native = _binding(backend)
    if native is not None and not _forward_ad_active() and native.paged_copy(
            key_cache, value_cache, sources, targets, tokens):
        return
    _check_backend(backend)
    _check_caches(key_cache, value_cache)
    pages, _, S, _ = key_cache.shape
    if S % _PAGE_MULTIPLE:
        raise ValueError(f"the page size must be a positive multiple of {_PAGE_MULTIPLE}; got {S}")
    _check_tensor("sources", sources, 1, "(pages to copy,)")
    n = sources.shape[0]
    for name, t in (("sources", sources), ("targets", targets), ("tokens", tokens)):
        if t is not None or name != "tokens":
            _check_ints(name, t, (n,), key_cache.device)
    if torch.is_grad_enabled() and (key_cache.requires_grad or value_cache.requires_grad):
        raise RuntimeError("paged_cache_copy records no gradients; call it under torch.no_grad()")
    if any(s == 0 and n > 1 for t in (key_cache, value_cache)
           for s, n in zip(t.stride(), t.shape)):
        raise ValueError("the caches must not be expanded tensors")
    if not torch.compiler.is_dynamo_compiling() and key_cache.data_ptr() == value_cache.data_ptr():
        raise ValueError("key_cache and value_cache must be different tensors")
    reason = None
    if backend != "torch":
        reason = (_gpu_reason(key_cache) if key_cache.device.type != "cuda"
                  else _cache_reason(key_cache, value_cache) or _gpu_reason(key_cache))
        if reason is None and key_cache[0].numel() >= 1 << 33:
            reason = "the pages are too large for one launch"
        elif reason is None and _forward_ad_active():
            reason = "the copying kernel moves no tangents"
    if _falls_back(backend, reason):
        kept = (sources >= 0) & (sources < pages) & (targets >= 0) & (targets < pages)
        source, target = sources[kept].long(), targets[kept].long()
        for cache in (key_cache, value_cache):
            moved = cache[source]
            if tokens is not None:
                first = torch.arange(S, device=cache.device) < tokens[kept][:, None]
                moved = torch.where(first[:, None, :, None], moved, cache[target])
            cache[target] = moved
        return
    if n:
        _ops.paged_copy(key_cache, value_cache, sources, targets, tokens)


# ---- compact ----------------------------------------------------------------------------


def _torch_compact(page_table, free_pages, page_shares, free_start):
    P, F, device = page_shares.shape[0], free_pages.shape[0], page_table.device
    start = _start(free_start, free_pages)
    place = torch.arange(F, device=device)
    named = (place >= start) & (free_pages >= 0) & (free_pages < P)
    held = torch.ones(P, dtype=torch.bool, device=device)
    held[free_pages[named].long()] = False
    page, used = torch.arange(P, device=device), held.sum()
    source = torch.nonzero(held & (page >= used)).squeeze(1)
    target = torch.nonzero(~held & (page < used)).squeeze(1)
    new = page.clone()
    new[source] = target
    entry = (page_table >= 0) & (page_table < P)
    table = torch.where(entry, new[torch.where(entry, page_table, 0).long()], page_table)
    shares = torch.where(held & (page < used), page_shares, 0)
    shares[target] = page_shares[source]
    free = used + place - start
    free = torch.where(place < start, free_pages, torch.where(free < P, free, -1))
    moves = torch.full((2, F), -1, dtype=torch.int32, device=device)
    moves[0, :source.shape[0]], moves[1, :source.shape[0]] = source.int(), target.int()
    return PagedCompaction(table.to(torch.int32), free.to(torch.int32), shares, moves[0], moves[1],
                           used.reshape(1).to(torch.int32))


def paged_cache_compact(
    page_table: torch.Tensor,
    free_pages: torch.Tensor,
    page_shares: torch.Tensor,
    *,
    free_start: torch.Tensor | None = None,
    backend: Backend = "auto",
) -> PagedCompaction:
    """The bookkeeping of a cache whose held pages move to its front, so that its end can be given
    back or taken by another.

    Held are the pages that ``free_pages`` [F] does not name from place ``free_start`` (0 by
    default, taken into [0, F]) on; there are ``used`` of them. The k-th held page from page
    ``used`` on, ``sources[k]``, moves to the k-th free page in front of it, ``targets[k]``; for
    every layer ``paged_cache_copy(key_cache, value_cache, c.sources, c.targets)`` moves it. The
    returned table names the new places in every entry that named a page that moves, the returned
    counts follow the pages (0 for free ones), and the returned list holds ``used``, ``used + 1``,
    ... from ``free_start`` on (-1 where it is longer). All integers are int32; the tensors passed
    in stay as they are, and a program that holds pages outside the table finds them in ``sources``.
    """
    native = _binding(backend)
    if native is not None:
        out = native.paged_compact(page_table, free_pages, page_shares, free_start)
        if out is not None:
            return PagedCompaction(*out)
    _check_backend(backend)
    _check_table(page_table, _PAGE_MULTIPLE)
    _check_lists(page_table, free_pages, page_shares, free_start)
    reason = None
    if backend != "torch":
        reason = _gpu_reason(page_table)
        if reason is None and (page_table.shape[0] >= 1 << 17
                               or max(free_pages.shape[0], page_shares.shape[0]) >= _MOST):
            reason = "too many sequences or pages for one launch"
    if _falls_back(backend, reason):
        return _torch_compact(page_table, free_pages, page_shares, free_start)
    return PagedCompaction(*_ops.paged_compact(page_table, free_pages, page_shares, free_start))
