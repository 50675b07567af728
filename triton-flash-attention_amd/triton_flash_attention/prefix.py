"""Attention over the paged cache where groups of sequences share a prefix (csrc/fa_prefix.hip):
the beams of a request over its prompt, samples of one prompt, requests that begin with the same
instructions or ask about the same document. The prefix's keys and values are read once for a
group and meet the queries of all its sequences as one matrix product.

No counterpart in the reference. Names, checks and the choice of a backend follow :mod:`.paged`.
"""

from __future__ import annotations

import math

import torch

from . import _ops
from .attention import Backend, _forward_ad_active
from .paged import (_attention_reason, _check_attention, _check_ints, _scaled_query)
from .rotary import _binding, _check_backend, _check_tensor, _falls_back

# Query rows of a tile: of a prefix, and of a sequence's own keys where it has at most _OWN_ROWS
# (fa_layer.hpp kPrefixTile, kOwnTile, kOwnRows).
_TILE, _OWN_TILE, _OWN_ROWS = 128, 32, 64


def _prefixes(lengths, group_starts, prefix_lengths, capacity):
    """(each sequence's prefix keys, the sequence whose pages hold them, whether the groups'
    starts ascend within the batch)."""
    B, G = lengths.shape[0], prefix_lengths.shape[0]
    starts, b = group_starts.long(), torch.arange(B, device=lengths.device)
    good = ((starts >= 0) & (starts <= B)).all() & (starts[1:] >= starts[:-1]).all()
    if G == 0:
        return torch.zeros_like(b), b, good
    g = (starts[None, :] <= b[:, None]).sum(1) - 1
    inside, g = (g >= 0) & (g < G), g.clamp(0, G - 1)
    first = starts[g].clamp(0, B - 1)
    held = lengths[first].long()
    held = torch.where(held <= capacity, held, 0)
    keys = torch.minimum(prefix_lengths[g].long(), held).clamp(min=0)
    return torch.where(good & inside & (starts[g + 1] - starts[g] >= 2), keys, 0), first, good


def _torch_prefix(query, key_cache, value_cache, page_table, lengths, group_starts, prefix_lengths,
                  scale):
    """The formulas in PyTorch, in float32 (float64 for float64 inputs), one sequence at a time."""
    wide = torch.float64 if query.dtype == torch.float64 else torch.float32
    B, Hq, N, D = query.shape
    pages, H, S, _ = key_cache.shape
    capacity = page_table.shape[1] * S
    at = torch.arange(capacity, device=query.device)
    keys, first, ascend = _prefixes(lengths, group_starts, prefix_lengths, capacity)
    out = []
    for b in range(B):
        length = lengths[b]
        fits = (length >= 0) & (length <= capacity) & ascend
        page = torch.where(at < keys[b], page_table[first[b]][at // S], page_table[b][at // S]).long()
        known = (page >= 0) & (page < pages)
        # what lies behind the length is no part of the sequence, whatever it holds
        inside = at < length
        good = fits & (known | ~inside).all()
        page = torch.where(known, page, 0)
        k, v = (torch.where(inside[:, None, None], t[page, :, at % S], 0).transpose(0, 1).to(wide)
                for t in (key_cache, value_cache))
        last = length - N + torch.arange(N, device=query.device)
        seen = (at[None, :] <= last[:, None]).repeat(Hq // H, 1)
        q = query[b].to(wide).reshape(H, Hq // H * N, D)
        scores = torch.matmul(q, k.transpose(1, 2).contiguous()) * scale
        scores = scores.masked_fill(~seen, -math.inf)
        m = scores.amax(-1, keepdim=True).detach()
        p = torch.exp(scores - torch.where(m == -math.inf, 0.0, m))
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p / torch.where(total == 0, 1.0, total), v.contiguous()).reshape(Hq, N, D)
        out.append(torch.where(good, o, math.nan))
    return torch.stack(out).to(query.dtype)


def paged_prefix_attention(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    group_starts: torch.Tensor,
    prefix_lengths: torch.Tensor,
    *,
    scale: float | None = None,
    enable_gqa: bool = False,
    backend: Backend = "auto",
) -> torch.Tensor:
    """Attention of the newest tokens of each sequence over the paged cache, with the keys that
    groups of sequences share read once for each group.

    query [B, Hq, N, D], the caches, ``page_table`` [B, M] and ``lengths`` [B] are those of
    :func:`.paged.paged_attention`, and so are the keys that a query sees and the rows that are 0
    or NaN. Group g of ``group_starts`` [G + 1] (int32) holds the sequences ``group_starts[g]`` to
    ``group_starts[g + 1] - 1``; sequences outside all groups share nothing. Its prefix is the
    first ``prefix_lengths[g]`` (int32) tokens of its first sequence, at most as many as this one
    holds: for all sequences of the group these keys and values lie in the first one's pages, so
    the entries of the others' rows of ``page_table`` for whole pages of it are not read. Where the
    prefix ends inside a page, the keys behind it are in each sequence's own page.

    ``group_starts`` that do not ascend from 0 or more to B or less make all rows NaN. A NaN or an
    infinity in the values of a prefix's token reaches all rows of its group, also those of a
    sequence that is shorter.

    The gfx950 kernels serve what those of ``paged_attention`` serve, in fewer than 2^24 groups, and
    have no backward. They work on tiles of 128 of the rows that share a prefix and a key/value head,
    and take about 15 us before the keys count. Where the rows of ``page_table`` name the shared pages
    themselves (as forks leave them), ``paged_attention`` gives the same rows, and sooner for short
    prefixes: with 32 query heads on 8 and D = 128, up to some 1000 shared keys (6 us against 16 at
    128), 2000 for four sequences and 8000 for two; over 8192 keys 32 sequences take 33 us here and
    84 there. For sequences that share nothing ``paged_attention`` is faster as well.
    """
    native = _binding(backend)
    if native is not None and not _forward_ad_active():
        out = native.paged_prefix_attention(query, key_cache, value_cache, page_table, lengths,
                                            group_starts, prefix_lengths, scale, enable_gqa)
        if out is not None:
            return out
    _check_backend(backend)
    _check_attention(query, key_cache, value_cache, page_table, lengths, scale, enable_gqa)
    B, Hq, N, D = query.shape
    H, S = key_cache.shape[1:3]
    _check_tensor("prefix_lengths", prefix_lengths, 1, "(groups,)")
    G = prefix_lengths.shape[0]
    _check_ints("prefix_lengths", prefix_lengths, (G,), query.device)
    _check_ints("group_starts", group_starts, (G + 1,), query.device)
    softmax_scale = float(scale) if scale is not None else D ** -0.5
    rows = Hq // H * N
    tiles = B * H * -(-rows // (_OWN_TILE if rows <= _OWN_ROWS else _TILE))
    if G > 0 and B > 1:
        tiles += H * (B * rows // _TILE + min(G, B // 2))
    too_many = Hq >= 1 << 20 or N >= 1 << 20 or G >= 1 << 24 or B * Hq * N >= 1 << 24 or (
        tiles * (-(-page_table.shape[1] * S // 32) + 24) >= 1 << 30)
    reason, served = _attention_reason(backend, query, key_cache, value_cache, softmax_scale, too_many)
    if _falls_back(backend, reason):
        return _torch_prefix(query, key_cache, value_cache, page_table, lengths, group_starts,
                             prefix_lengths, softmax_scale)
    query, kernel_scale = _scaled_query(query, served)
    return _ops.paged_prefix_fwd(query, key_cache, value_cache, page_table, lengths, group_starts,
                                 prefix_lengths, kernel_scale)
