"""Attention over shared prefixes where its work spreads over the whole chip: rows of thousands of
pieces, prefixes that are cut into pieces, and the memory that a call may write."""

from __future__ import annotations

import pytest
import torch
from test_paged import F32, HALF
from test_prefix import within

from triton_flash_attention import paged_prefix_attention


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize(("D", "n"), [(32, 262144), (64, 262144), (64, 1 << 20), (128, 262144)])
def test_join_of_thousands_of_pieces_keeps_values_near_the_largest(D, n, shared):
    """One key head and a sequence that holds nearly all keys of the call: with equal scores its row is
    the mean of 2048 to 2979 pieces of up to 3.3e38 each, near the largest float32. The mean of n values
    of at most A is off by the roundings of the output and of the 16-bit probabilities, which are equal,
    and by the additions in a piece (of fewer than n / 2048 + 64 keys) and of 3840 pieces at most."""
    S, Hq, dtype = 64, 2, torch.bfloat16
    gen = torch.Generator("cuda").manual_seed(D)
    pages = n // S + 1
    k = torch.zeros(pages, 1, S, D, dtype=dtype, device="cuda")
    v = (2.0 + 1.8 * torch.rand(pages, 1, S, D, generator=gen, device="cuda")).to(dtype)
    v = v * 2.0 ** 126
    lengths = [n + 1, 7] if shared else [n, 7]
    table = torch.zeros(2, pages, dtype=torch.int32, device="cuda")
    table[0] = torch.randperm(pages, generator=gen, device="cuda").int()
    q = torch.randn(2, Hq, 1, D, generator=gen, device="cuda").to(dtype)
    groups = (ints([0, 2]), ints([5])) if shared else (ints([0]), ints([]))
    o = paged_prefix_attention(q, k, v, table, ints(lengths), *groups, enable_gqa=True,
                               backend="triton")
    rows = v[table[0].long(), 0].double().reshape(-1, D)[:lengths[0]]
    want = rows.mean(0).expand(Hq, 1, D).cpu()
    bound = want * (HALF[dtype] + (n // 2048 + 64 + 3840) * F32)
    within(o[0], want, bound, dtype)
