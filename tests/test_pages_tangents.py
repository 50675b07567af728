"""Forward-mode derivatives of the calls that write the paged cache: caches with tangents keep them where
they were written, on the CPU and beside the gfx950 kernels."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD
from test_pages import ints

from triton_flash_attention import paged_cache_copy, paged_cache_store


def dual_caches(device, pages=5, H=2, S=16, D=32):
    gen = torch.Generator().manual_seed(4)
    t = [torch.randn(pages, H, S, D, generator=gen).half().to(device) for _ in range(4)]
    return t[:2], t[2:]


def check_copy_tangents(device, backend, tokens):
    primals, tangents = dual_caches(device)
    want = [t.clone() for t in (*primals, *tangents)]
    rows = 16 if tokens is None else tokens
    for w in want:
        w[1, :, :rows] = w[3, :, :rows]
    with fwAD.dual_level():
        caches = [fwAD.make_dual(p.clone(), t.clone()) for p, t in zip(primals, tangents)]
        paged_cache_copy(*caches, ints([3, -1], device), ints([1, 0], device),
                         tokens=None if tokens is None else ints([tokens, 0], device), backend=backend)
        got = [fwAD.unpack_dual(c) for c in caches]
        assert all(torch.equal(g.primal, w) for g, w in zip(got, want[:2]))
        assert all(torch.equal(g.tangent, w) for g, w in zip(got, want[2:]))


@pytest.mark.parametrize("tokens", [None, 5])
def test_copy_moves_tangents(tokens):
    check_copy_tangents("cpu", "auto", tokens)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [None, 5])
def test_copy_moves_tangents_on_the_gpu(tokens):
    check_copy_tangents("cuda", "auto", tokens)
    with fwAD.dual_level(), pytest.raises(RuntimeError, match="no tangents"):
        primals, tangents = dual_caches("cuda")
        paged_cache_copy(*map(fwAD.make_dual, primals, tangents), ints([3], "cuda"), ints([1], "cuda"),
                         backend="triton")
    primals, _ = dual_caches("cuda")  # outside a level the kernel serves the call as before
    paged_cache_copy(*primals, ints([3], "cuda"), ints([1], "cuda"), backend="triton")
    assert all(torch.equal(p[1], p[3]) for p in primals)


def check_store_tangents(device, backend, dual_cache):
    """New tokens with tangents, into caches that have some or none yet."""
    primals, tangents = dual_caches(device)
    if not dual_cache:
        tangents = [torch.zeros_like(t) for t in tangents]
    gen = torch.Generator().manual_seed(5)
    new = [torch.randn(3, 2, 32, generator=gen).half().to(device) for _ in range(4)]
    want = [t.clone() for t in (*primals, *tangents)]
    for w, t in zip(want, new):
        w[2, :, 7], w[0, :, 15] = t[0], t[2]
    slots = torch.tensor([2 * 16 + 7, -1, 15], device=device)
    with fwAD.dual_level():
        caches = [fwAD.make_dual(p.clone(), t.clone()) if dual_cache else p.clone()
                  for p, t in zip(primals, tangents)]
        paged_cache_store(*map(fwAD.make_dual, new[:2], new[2:]), *caches, slots, backend=backend)
        got = [fwAD.unpack_dual(c) for c in caches]
        assert all(torch.equal(g.primal, w) for g, w in zip(got, want[:2]))
        assert all(torch.equal(g.tangent, w) for g, w in zip(got, want[2:]))


@pytest.mark.parametrize("dual_cache", [True, False])
def test_store_writes_tangents(dual_cache):
    check_store_tangents("cpu", "auto", dual_cache)


@pytest.mark.gpu
@pytest.mark.parametrize("dual_cache", [True, False])
def test_store_writes_tangents_on_the_gpu(dual_cache):
    check_store_tangents("cuda", "auto", dual_cache)
    with pytest.raises(RuntimeError, match="no tangents"):
        check_store_tangents("cuda", "triton", dual_cache)
