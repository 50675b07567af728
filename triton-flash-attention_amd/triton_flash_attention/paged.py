"""The paged key/value cache of a serving program: the plan of a step (which pages and slots
its new tokens take), the store of their keys and values, and the attention of new tokens over
the cache (csrc/fa_paged.hip).

The cache is two tensors [pages, Hkv, page_size, D] that the program allocates once; a page
holds ``page_size`` tokens (a multiple of 16) of one sequence, and row b of the page table
[B, M] names the pages of sequence b in order. Lengths, tables and slots stay on the GPU: the
kernels' calls read none of them on the host, so a decoding step can be captured into a graph
(the PyTorch forms of the plan and the store do read them). What they hold is checked on the GPU.

A step of T tokens, q [1, Hq, T, D], k and v [1, Hkv, T, D], of which each sequence's newest n
are attended (``starts`` says where a sequence's tokens end; when decoding, T = B and n = 1):

    plan = paged_cache_plan(table, lengths, new_tokens, free_pages, page_size=16, num_tokens=T)
    q, k = qk_norm_rope(q, k, cos, sin, positions=plan.positions)
    paged_cache_store(k[0].transpose(0, 1), v[0].transpose(0, 1), key_cache, value_cache,
                      plan.slots)
    newest = plan.starts[1:, None] - n + torch.arange(n, device=q.device)
    q = q[0][:, newest].transpose(0, 1)  # [B, Hq, n, D]
    out = paged_attention(q, key_cache, value_cache, table, plan.lengths, enable_gqa=True)

No counterpart in the reference, which attends over dense [B, H, N, D] tensors. Names, checks
and the choice of a backend follow :mod:`.attention`.
"""

from __future__ import annotations

import math
from numbers import Real
from typing import NamedTuple

import torch

from . import _ops
from .attention import _SUPPORTED_DTYPES, Backend, _forward_ad_active, _kernel_scale
from .rotary import _binding, _check_backend, _check_tensor, _falls_back, _gpu_reason

_PAGE_MULTIPLE = 16
_MOST_TOKENS = (1 << 30) - 64  # that a row of the page table holds (fa_capi_layer.hip)


class PagedPlan(NamedTuple):
    """Where a step's new tokens go (:func:`paged_cache_plan`)."""

    slots: torch.Tensor       # [num_tokens] int64, page * page_size + row; -1 for no slot
    positions: torch.Tensor   # [num_tokens] int32, each token's place in its sequence
    starts: torch.Tensor      # [B + 1] int32, each sequence's first token in the step
    lengths: torch.Tensor     # [B] int32, tokens held after the step
    free_start: torch.Tensor  # [1] int32, place of the first page that stays free


def _check_ints(name: str, t, shape: tuple, device) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}; got {tuple(t.shape)}")
    if t.dtype != torch.int32 or t.device != device:
        raise ValueError(f"{name} must be int32 on {device}")


def _check_table(page_table, page_size) -> None:
    _check_tensor("page_table", page_table, 2, "(batch, pages)")
    if page_table.dtype != torch.int32:
        raise ValueError(f"page_table must be int32; got {page_table.dtype}")
    if page_table.shape[1] == 0:
        raise ValueError("page_table must have at least one column")
    if isinstance(page_size, bool) or not isinstance(page_size, int) or page_size <= 0 or (
            page_size % _PAGE_MULTIPLE):
        raise ValueError(
            f"the page size must be a positive multiple of {_PAGE_MULTIPLE}; got {page_size!r}")
    if page_table.shape[1] * page_size > _MOST_TOKENS:
        raise ValueError(f"page_table holds more than {_MOST_TOKENS} tokens a sequence")


def _check_caches(key_cache, value_cache) -> None:
    for name, t in (("key_cache", key_cache), ("value_cache", value_cache)):
        _check_tensor(name, t, 4, "(pages, heads, page_size, head_dim)")
        if 0 in t.shape:
            raise ValueError(f"{name} dimensions must all be greater than zero")
    if key_cache.shape != value_cache.shape:
        raise ValueError("key_cache and value_cache must have the same shape")
    if key_cache.device != value_cache.device or key_cache.dtype != value_cache.dtype:
        raise ValueError("key_cache and value_cache must share a device and a dtype")


def _cache_reason(key_cache, value_cache) -> str | None:
    """Why the kernels cannot address these caches (as they stand: they are not copied)."""
    if key_cache.dtype not in _SUPPORTED_DTYPES:
        return "the kernel currently supports float16 and bfloat16"
    if key_cache.shape[3] > 128 or key_cache.shape[3] % 8:
        return "head_dim must be a multiple of 8 of at most 128"
    strides = _ops.cache_strides(key_cache)
    if strides != _ops.cache_strides(value_cache):
        return "key_cache and value_cache must have the same strides"
    if any(t.stride(3) != 1 or t.data_ptr() % 16 or t.is_neg() for t in (key_cache, value_cache)) or (
            any(s % 8 for s in strides)):
        return "the caches' rows must be contiguous, 16-byte aligned and a multiple of 8 apart"
    if not key_cache.shape[3] <= strides[2] < 1 << 25 or max(strides) >= 1 << 40 or (
            key_cache.shape[0] >= 1 << 31):
        return "the caches' strides are outside the kernel's addressing"
    return None


# ---- plan -------------------------------------------------------------------------------


def _torch_plan(page_table, lengths, new_tokens, free_pages, free_start, page_size, num_tokens):
    S, (B, M), F = page_size, page_table.shape, free_pages.shape[0]
    device, most = page_table.device, (1 << 30) - 1
    held_tokens, new = (t.long().clamp(0, most) for t in (lengths, new_tokens))
    held = (held_tokens + S - 1) // S
    need = (((held_tokens + new + S - 1) // S).clamp(max=M) - held).clamp(min=0)
    ends = torch.cumsum(new, 0)
    zero = torch.zeros(1, dtype=torch.int64, device=device)
    starts = torch.cat((zero, ends))
    first = zero if free_start is None else free_start.reshape(1).long()
    places = first + torch.cat((zero, torch.cumsum(need, 0)))
    t = torch.arange(num_tokens, device=device)
    slots = torch.full((num_tokens,), -1, dtype=torch.int64, device=device)
    positions = torch.zeros(num_tokens, dtype=torch.int32, device=device)
    if B and num_tokens:
        row = torch.searchsorted(ends, t, right=True).clamp(max=B - 1)
        real = t < ends[-1]
        position = torch.where(real, held_tokens[row] + t - starts[row], 0)
        j = position // S
        place = places[row] + j - held[row]
        fresh = real & (j >= held[row]) & (j < M)
        supplied = fresh & (place >= 0) & (place < F)
        page = page_table[row, j.clamp(max=M - 1)].long()
        if F:
            new_page = free_pages[place.clamp(0, F - 1)].long()
            page = torch.where(fresh, torch.where(supplied, new_page, -1), page)
        else:
            page = torch.where(fresh, -1, page)
        opens = fresh & (position % S == 0)
        page_table[row[opens], j[opens]] = page[opens].to(torch.int32)
        page = torch.where(real & (j < M), page, -1)
        slots = torch.where(page >= 0, page * S + position % S, -1)
        positions = position.to(torch.int32)
    small = (1 << 31) - 1
    return PagedPlan(slots, positions, starts.clamp(max=small).to(torch.int32),
                     (held_tokens + new).to(torch.int32),
                     places[-1:].clamp(0, small).to(torch.int32))


def paged_cache_plan(
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    new_tokens: torch.Tensor,
    free_pages: torch.Tensor,
    *,
    page_size: int,
    num_tokens: int,
    free_start: torch.Tensor | None = None,
    backend: Backend = "auto",
) -> PagedPlan:
    """Pages and slots of a step's new tokens, from the sequences' lengths.

    Sequence b holds ``lengths[b]`` tokens in the pages of row b of ``page_table`` [B, M] and
    gets ``new_tokens[b]`` more. The pages that these open are taken from ``free_pages`` in the
    order of the sequences, from place ``free_start`` (a tensor of one value; 0 by default) on,
    and written into the table in place, which changes no other entry. The tokens of the step
    are numbered in the order of the sequences; ``num_tokens`` (an upper bound the program
    knows, at least their number) is the length of the returned ``slots`` and ``positions``,
    whose rows behind the last token hold slot -1 and position 0. All integers are int32.

    Where the free pages do not suffice, the missing table entries and their tokens' slots are
    -1 and ``free_start`` of the result exceeds ``len(free_pages)``; tokens behind a sequence's
    M pages have slot -1 as well. Negative lengths and counts are taken as 0.
    """
    native = _binding(backend)
    if native is not None:
        out = native.paged_plan(page_table, lengths, new_tokens, free_pages, page_size, num_tokens,
                                free_start)
        if out is not None:
            return PagedPlan(*out)
    _check_backend(backend)
    _check_table(page_table, page_size)
    B, device = page_table.shape[0], page_table.device
    for name, t in (("lengths", lengths), ("new_tokens", new_tokens)):
        _check_ints(name, t, (B,), device)
    _check_tensor("free_pages", free_pages, 1, "(free pages,)")
    _check_ints("free_pages", free_pages, tuple(free_pages.shape), device)
    if free_start is not None:
        _check_tensor("free_start", free_start, free_start.ndim if isinstance(
            free_start, torch.Tensor) else 1, "(1,)")
        if free_start.numel() != 1 or free_start.dtype != torch.int32 or free_start.device != device:
            raise ValueError(f"free_start must be one int32 value on {device}")
    if isinstance(num_tokens, bool) or not isinstance(num_tokens, int) or not (
            0 <= num_tokens < 1 << 30):
        raise ValueError(f"num_tokens must be an int from 0 to 2^30 - 1; got {num_tokens!r}")
    if B > 1 and page_table.stride(0) < page_table.shape[1]:
        raise ValueError("the rows of page_table must not overlap")
    reason = None
    if backend != "torch":
        reason = _gpu_reason(page_table)
        if reason is None and page_table.stride(1) != 1 and page_table.shape[1] > 1:
            reason = "the rows of page_table must be contiguous"
    if _falls_back(backend, reason):
        return _torch_plan(page_table, lengths, new_tokens, free_pages, free_start, page_size,
                           num_tokens)
    return PagedPlan(*_ops.paged_plan(page_table, lengths, new_tokens, free_pages, free_start,
                                      page_size, num_tokens))


# ---- store ------------------------------------------------------------------------------


def paged_cache_store(
    key: torch.Tensor,
    value: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    slots: torch.Tensor,
    *,
    backend: Backend = "auto",
) -> None:
    """Write the keys and values of new tokens into their slots of the cache, in place.

    key and value are [T, Hkv, D], views allowed (``k.transpose(1, 2).flatten(0, 1)`` of a
    [B, Hkv, N, D] tensor); ``slots`` [T] (int64) as :func:`paged_cache_plan` returns them:
    slot s is row ``s % page_size`` of page ``s // page_size``. Negative slots and slots behind
    the last page are left out; the others must differ from each other. Rows of the cache that
    no slot names stay as they were. key and value must not share memory with the cache.
    Gradients are not recorded: the call raises where one would have to be.
    """
    native = _binding(backend)
    if native is not None and native.paged_store(key, value, key_cache, value_cache, slots):
        return
    _check_backend(backend)
    for name, t in (("key", key), ("value", value)):
        _check_tensor(name, t, 3, "(tokens, heads, head_dim)")
    if key.shape != value.shape:
        raise ValueError("key and value must have the same shape")
    _check_caches(key_cache, value_cache)
    pages, H, S, D = key_cache.shape
    if S % _PAGE_MULTIPLE:
        raise ValueError(f"the page size must be a positive multiple of {_PAGE_MULTIPLE}; got {S}")
    if tuple(key.shape[1:]) != (H, D):
        raise ValueError(f"key and value must have shape (tokens, {H}, {D}); got {tuple(key.shape)}")
    if not isinstance(slots, torch.Tensor):
        raise TypeError("slots must be a torch.Tensor")
    if tuple(slots.shape) != (key.shape[0],) or slots.dtype != torch.int64:
        raise ValueError(f"slots must have shape ({key.shape[0]},) and be int64")
    tensors = (key, value, key_cache, value_cache)
    if any(t.device != key_cache.device for t in (*tensors, slots)):
        raise ValueError("key, value, the caches and slots must be on the same device")
    if key.dtype != key_cache.dtype or value.dtype != key_cache.dtype:
        raise ValueError("key, value and the caches must have the same dtype")
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError("paged_cache_store records no gradients; call it under torch.no_grad()")
    if any(s == 0 and n > 1 for t in (key_cache, value_cache)
           for s, n in zip(t.stride(), t.shape)):
        raise ValueError("the caches must not be expanded tensors")
    if not torch.compiler.is_dynamo_compiling() and key_cache.data_ptr() == value_cache.data_ptr():
        raise ValueError("key_cache and value_cache must be different tensors")
    reason = None
    if backend != "torch":
        reason = (_gpu_reason(key_cache) if key_cache.device.type != "cuda"
                  else _cache_reason(key_cache, value_cache) or _gpu_reason(key_cache))
    if _falls_back(backend, reason):
        kept = torch.nonzero((slots >= 0) & (slots < pages * S)).squeeze(1)
        page, row = slots[kept] // S, slots[kept] % S
        key_cache[page, :, row] = key[kept]
        value_cache[page, :, row] = value[kept]
        return
    if key.shape[0]:
        _ops.paged_store(key, value, key_cache, value_cache, slots)


# ---- attention --------------------------------------------------------------------------


def _torch_paged(query, key_cache, value_cache, page_table, lengths, scale):
    """The formulas in PyTorch, in float32 (float64 for float64 inputs), one sequence at a time."""
    wide = torch.float64 if query.dtype == torch.float64 else torch.float32
    B, Hq, N, D = query.shape
    pages, H, S, _ = key_cache.shape
    capacity = page_table.shape[1] * S
    at = torch.arange(capacity, device=query.device)
    out = []
    for b in range(B):
        length, table = lengths[b], page_table[b]
        fits = (length >= 0) & (length <= capacity)
        known = (table >= 0) & (table < pages)
        held = torch.arange(table.shape[0], device=query.device) * S < length
        good = fits & (known | ~held).all()
        chosen = torch.where(known, table, 0).long()
        # what lies behind the length is no part of the sequence, whatever it holds
        inside = (at < length)[:, None]
        k, v = (torch.where(inside, t[chosen].transpose(0, 1).reshape(H, capacity, D), 0).to(wide)
                for t in (key_cache, value_cache))
        last = length - N + torch.arange(N, device=query.device)
        seen = (at[None, :] <= last[:, None]).repeat(Hq // H, 1)
        q = query[b].to(wide).reshape(H, Hq // H * N, D)
        scores = torch.matmul(q, k.transpose(1, 2).contiguous()) * scale
        scores = scores.masked_fill(~seen, -math.inf)
        m = scores.amax(-1, keepdim=True).detach()
        p = torch.exp(scores - torch.where(m == -math.inf, 0.0, m))
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p / torch.where(total == 0, 1.0, total), v).reshape(Hq, N, D)
        out.append(torch.where(good, o, math.nan))
    return torch.stack(out).to(query.dtype)


def _row_blocks(rows: int) -> int:
    """Passes over a key/value head's keys that its query rows take (fa_layer.hpp paged_rows)."""
    return 1 if rows <= 32 else -(-rows // 32)


def paged_attention(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    scale: float | None = None,
    enable_gqa: bool = False,
    backend: Backend = "auto",
) -> torch.Tensor:
    """Attention of the newest tokens of each sequence over the paged cache.

    query [B, Hq, N, D] holds the N newest tokens of each sequence (one when decoding, a few
    when drafted tokens are checked; strided views allowed), whose keys and values are in the
    cache already: ``lengths`` [B] (int32) counts them. Query n sees the keys
    ``j <= lengths[b] - N + n``, so the last one sees all. Returns the contiguous output
    [B, Hq, N, D].

    Rows that see no key are 0. A sequence whose length is negative or above what its row of
    ``page_table`` [B, M] (int32) holds, or that needs a page that is not in the cache, gets NaN.
    Table entries behind a sequence's length are not read, nor are the cache's rows there.
    A NaN or an infinity in the values of one of the N newest tokens reaches the earlier ones'
    rows too.

    The gfx950 kernel serves float16 and bfloat16 with head_dim a multiple of 8 up to 128. It
    reads the cache once for each 32 of the Hq / Hkv * N rows that share a key/value head, so it
    is made for one token or a few, not for a prompt's. Where a row of the table holds more than
    1024 keys (2048 where B * Hkv is 256 or more) the keys are split over the whole GPU whatever
    the lengths are; in a narrower table one work-group takes each of B * Hkv heads, which is
    faster for short sequences. It has no backward: inputs that require gradients run in PyTorch
    under ``backend="auto"``.
    """
    native = _binding(backend)
    if native is not None and not _forward_ad_active():
        out = native.paged_attention(query, key_cache, value_cache, page_table, lengths, scale,
                                     enable_gqa)
        if out is not None:
            return out
    _check_backend(backend)
    if not isinstance(enable_gqa, bool):
        raise TypeError("enable_gqa must be a bool")
    if scale is not None and (not isinstance(scale, Real) or not math.isfinite(float(scale))):
        raise ValueError("scale must be a finite real number or None")
    _check_tensor("query", query, 4, "(batch, heads, sequence, head_dim)")
    if 0 in query.shape:
        raise ValueError("query dimensions must all be greater than zero")
    _check_caches(key_cache, value_cache)
    B, Hq, N, D = query.shape
    H, S = key_cache.shape[1:3]
    _check_table(page_table, S)
    if query.device != key_cache.device or page_table.device != query.device:
        raise ValueError("query, the caches, page_table and lengths must be on the same device")
    if query.dtype != key_cache.dtype:
        raise ValueError("query and the caches must have the same dtype")
    if key_cache.shape[3] != D:
        raise ValueError("query and cache head dimensions must match")
    if page_table.shape[0] != B:
        raise ValueError("page_table must have a row for each sequence of query")
    _check_ints("lengths", lengths, (B,), query.device)
    if Hq != H and not enable_gqa:
        raise ValueError(
            "query has a different number of heads from key/value; pass "
            "enable_gqa=True to use grouped-query attention")
    if Hq % H:
        raise ValueError(
            "the number of query heads must be divisible by the number of key/value heads")
    softmax_scale = float(scale) if scale is not None else D ** -0.5
    reason = served = None
    if backend != "torch":
        if query.device.type != "cuda":
            reason = _gpu_reason(query)
        elif (served := _kernel_scale(softmax_scale)) is None:
            reason = f"scale {softmax_scale!r} overflows the gfx950 kernel's float32 arithmetic"
        elif _forward_ad_active() or (torch.is_grad_enabled() and any(
                t.requires_grad for t in (query, key_cache, value_cache))):
            reason = "the paged kernel has no backward"
        elif Hq >= 1 << 20 or N >= 1 << 20 or B * H * _row_blocks(Hq // H * N) * (
                -(-page_table.shape[1] * S // 32) + 24) >= 1 << 30:
            reason = "too many sequences, heads or keys for one launch"
        else:
            reason = _cache_reason(key_cache, value_cache) or _gpu_reason(query)
    if _falls_back(backend, reason):
        return _torch_paged(query, key_cache, value_cache, page_table, lengths, softmax_scale)
    kernel_scale, mode = served
    if mode == "negate":  # (-q).k |scale|
        query = -query
    elif mode == "zero":
        query = torch.zeros_like(query)
    return _ops.paged_fwd(query, key_cache, value_cache, page_table, lengths, kernel_scale)
