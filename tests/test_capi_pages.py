"""The C ABI of the operators on shared pages: arguments that are rejected before any HIP call (no GPU
needed; the fake addresses are never dereferenced)."""

from __future__ import annotations

import pytest
from test_capi_layer import P, ints, lib, rejected  # noqa: F401 - lib is a fixture

from triton_flash_attention import _lib


def prefix(lib, name="fa_paged_prefix_fwd", ws=P, ws_bytes=1 << 40, **change):  # noqa: F811
    a = dict(q=P, k=P, v=P, table=P, lengths=P, starts=P, prefix=P, o=P,
             strides=(256, 64, 64, 2048, 1024, 64, 100), B=2, G=1, Hq=4, Hkv=2, N=1, D=64, pages=4,
             M=100, S=16, scale=0.125)
    a.update(change)
    v = list(a.values())
    strides = None if v[8] is None else ints(*v[8])
    return getattr(lib, name)(*v[:8], strides, *v[9:], ws, ws_bytes, None)


@pytest.mark.parametrize(("change", "code", "message"), [
    (dict(q=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(starts=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(prefix=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(strides=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(ws=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(ws_bytes=1000), "FA_ERR_BAD_SHAPE", "smaller than"),
    (dict(G=-1), "FA_ERR_BAD_SHAPE", "negative"),
    (dict(Hq=3), "FA_ERR_BAD_SHAPE", "divisible"),
    (dict(N=0), "FA_ERR_BAD_SHAPE", "positive"),
    (dict(B=0), "FA_ERR_BAD_SHAPE", "positive"),
    (dict(D=132), "FA_ERR_HEAD_DIM", "multiple of 8"),
    (dict(S=12), "FA_ERR_BAD_SHAPE", "page size"),
    (dict(M=0), "FA_ERR_BAD_SHAPE", "columns"),
    (dict(pages=0), "FA_ERR_BAD_SHAPE", "pages"),
    (dict(G=1 << 30), "FA_ERR_TOO_LARGE", "too many"),
    (dict(N=1 << 25), "FA_ERR_TOO_LARGE", "too"),
    (dict(B=1 << 20, M=1 << 16), "FA_ERR_TOO_LARGE", "too many"),
    (dict(o=P + 4), "FA_ERR_MISALIGNED", "16-byte"),
    (dict(ws=P + 8), "FA_ERR_MISALIGNED", "16-byte"),
    (dict(starts=P + 2), "FA_ERR_MISALIGNED", "4-byte"),
    (dict(prefix=P + 1), "FA_ERR_MISALIGNED", "4-byte"),
    (dict(scale=0.0), "FA_ERR_BAD_SCALE", "scale"),
    (dict(scale=float("nan")), "FA_ERR_BAD_SCALE", "scale"),
    (dict(strides=(256, 64, 4, 2048, 1024, 64, 100)), "FA_ERR_BAD_STRIDE", "the query"),
    (dict(strides=(256, 64, 64, 2048, 1024, 32, 100)), "FA_ERR_BAD_STRIDE", "row stride"),
    (dict(strides=(256, 64, 64, 2048, 1024, 64, -1)), "FA_ERR_BAD_STRIDE", "page table"),
])
@pytest.mark.parametrize("name", ["fa_paged_prefix_fwd", "fa_paged_prefix_fwd_bf16"])
def test_prefix_rejects(lib, name, change, code, message):  # noqa: F811
    rejected(prefix(lib, name, **change), code, message)
    assert name in _lib.last_error()


def test_prefix_workspace(lib):  # noqa: F811
    need = lib.fa_paged_prefix_fwd_workspace_bytes(2, 1, 4, 2, 1, 64, 100, 16)
    assert need > 0 and need % 4 == 0
    rejected(prefix(lib, ws_bytes=need - 1), "FA_ERR_BAD_SHAPE", "smaller than")
    rejected(lib.fa_paged_prefix_fwd_workspace_bytes(2, -1, 4, 2, 1, 64, 100, 16), "FA_ERR_BAD_SHAPE",
             "negative")
    rejected(lib.fa_paged_prefix_fwd_workspace_bytes(2, 1, 4, 3, 1, 64, 100, 16), "FA_ERR_BAD_SHAPE",
             "divisible")


def fork(lib, ws=P, ws_bytes=1 << 30, **change):  # noqa: F811
    a = dict(table=P, table_stride=4, lengths=P, parents=P, free=P, start=None, shares=P, lengths_out=P,
             sources=P, targets=P, tokens=P, free_out=P, B=2, M=4, S=16, F=8, pages=8)
    a.update(change)
    return lib.fa_paged_fork(*a.values(), ws, ws_bytes, None)


@pytest.mark.parametrize(("change", "code", "message"), [
    (dict(S=0), "FA_ERR_BAD_SHAPE", "page size"),
    (dict(S=40), "FA_ERR_BAD_SHAPE", "page size"),
    (dict(M=0), "FA_ERR_BAD_SHAPE", "columns"),
    (dict(B=-1), "FA_ERR_BAD_SHAPE", "negative"),
    (dict(F=-1), "FA_ERR_BAD_SHAPE", "negative"),
    (dict(pages=0), "FA_ERR_BAD_SHAPE", "positive"),
    (dict(B=1 << 17), "FA_ERR_TOO_LARGE", "too many"),
    (dict(pages=1 << 30), "FA_ERR_TOO_LARGE", "too many"),
    (dict(F=1 << 30), "FA_ERR_TOO_LARGE", "too many"),
    (dict(table=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(parents=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(free=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(shares=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(free_out=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(ws=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(ws_bytes=0), "FA_ERR_BAD_SHAPE", "smaller than"),
    (dict(tokens=P + 2), "FA_ERR_MISALIGNED", "4-byte"),
    (dict(start=P + 1), "FA_ERR_MISALIGNED", "4-byte"),
    (dict(table_stride=3), "FA_ERR_BAD_STRIDE", "overlap"),
    (dict(B=1, table_stride=-1), "FA_ERR_BAD_STRIDE", "overlap"),
])
def test_fork_rejects(lib, change, code, message):  # noqa: F811
    rejected(fork(lib, **change), code, message)


def copy(lib, **change):  # noqa: F811
    a = dict(k=P, v=P, sources=P, targets=P, tokens=None, strides=(2048, 1024, 64), n=3, H=2, D=64,
             pages=4, S=16)
    a.update(change)
    v = list(a.values())
    return lib.fa_paged_copy(*v[:5], None if v[5] is None else ints(*v[5]), *v[6:], None)


@pytest.mark.parametrize(("change", "code", "message"), [
    (dict(k=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(targets=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(strides=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(n=-1), "FA_ERR_BAD_SHAPE", "positive"),
    (dict(H=0), "FA_ERR_BAD_SHAPE", "positive"),
    (dict(D=4), "FA_ERR_HEAD_DIM", "multiple of 8"),
    (dict(S=8), "FA_ERR_BAD_SHAPE", "page size"),
    (dict(pages=0), "FA_ERR_BAD_SHAPE", "pages"),
    (dict(n=1 << 31), "FA_ERR_TOO_LARGE", "too many"),
    (dict(H=1 << 19, S=1 << 12), "FA_ERR_TOO_LARGE", "too large"),
    (dict(v=P + 8), "FA_ERR_MISALIGNED", "16-byte"),
    (dict(sources=P + 2), "FA_ERR_MISALIGNED", "4-byte"),
    (dict(tokens=P + 1), "FA_ERR_MISALIGNED", "4-byte"),
    (dict(strides=(2048, 1024, 56)), "FA_ERR_BAD_STRIDE", "row stride"),
    (dict(strides=(2048, 1024, 1 << 25)), "FA_ERR_BAD_STRIDE", "row stride"),
])
def test_copy_rejects(lib, change, code, message):  # noqa: F811
    rejected(copy(lib, **change), code, message)


def test_copy_of_no_pages_is_no_launch(lib):  # noqa: F811
    assert copy(lib, n=0, k=None) == _lib.FA_OK


def compact(lib, ws=P, ws_bytes=1 << 30, **change):  # noqa: F811
    a = dict(table=P, table_stride=4, free=P, start=None, shares=P, table_out=P, free_out=P,
             shares_out=P, sources=P, targets=P, used=P, B=2, M=4, F=8, pages=8)
    a.update(change)
    return lib.fa_paged_compact(*a.values(), ws, ws_bytes, None)


@pytest.mark.parametrize(("change", "code", "message"), [
    (dict(M=0), "FA_ERR_BAD_SHAPE", "positive"),
    (dict(pages=0), "FA_ERR_BAD_SHAPE", "positive"),
    (dict(B=-1), "FA_ERR_BAD_SHAPE", "negative"),
    (dict(B=1 << 17), "FA_ERR_TOO_LARGE", "too many"),
    (dict(pages=1 << 30), "FA_ERR_TOO_LARGE", "too many"),
    (dict(table=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(free_out=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(used=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(ws=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(ws=P + 4), "FA_ERR_MISALIGNED", "16-byte"),
    (dict(ws_bytes=0), "FA_ERR_BAD_SHAPE", "smaller than"),
    (dict(shares_out=P + 2), "FA_ERR_MISALIGNED", "4-byte"),
    (dict(table_stride=-1), "FA_ERR_BAD_STRIDE", "negative"),
])
def test_compact_rejects(lib, change, code, message):  # noqa: F811
    rejected(compact(lib, **change), code, message)


def test_pages_workspaces(lib):  # noqa: F811
    need = lib.fa_paged_fork_workspace_bytes(2, 4, 8)
    assert need > 0
    rejected(fork(lib, ws_bytes=need - 1), "FA_ERR_BAD_SHAPE", "smaller than")
    need = lib.fa_paged_compact_workspace_bytes(8)
    assert need > 0
    rejected(compact(lib, ws_bytes=need - 1), "FA_ERR_BAD_SHAPE", "smaller than")
    rejected(lib.fa_paged_fork_workspace_bytes(2, 4, 0), "FA_ERR_BAD_SHAPE", "positive")
    rejected(lib.fa_paged_compact_workspace_bytes(0), "FA_ERR_BAD_SHAPE", "positive")
