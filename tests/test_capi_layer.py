"""The C ABI of the operators around the attention call: arguments that are rejected before any
HIP call (no GPU needed; the fake addresses are never dereferenced)."""

from __future__ import annotations

import ctypes

import pytest

from triton_flash_attention import _lib

P = 0x10000


@pytest.fixture(scope="module")
def lib():
    ok, why = _lib.available()
    assert ok, why
    return _lib.load()


def ints(*v):
    return (ctypes.c_int64 * len(v))(*v)


def rejected(rc, code, message):
    assert rc == getattr(_lib, code), (rc, _lib.last_error())
    assert message in _lib.last_error(), _lib.last_error()


# q, k: [2, 4 and 2, 8, 64] contiguous; positions [2, 8]
ROPE = dict(q=P, k=P, q_out=P, k_out=P, cos=P, sin=P, positions=P, q_weight=P, k_weight=P,
            strides=(2048, 512, 64, 1024, 512, 64, 8, 1), B=2, Hq=4, Hkv=2, N=8, D=64, R=64, P=8,
            eps=1e-6, flags=0)


def rope(lib, name="fa_qk_norm_rope", **change):
    a = {**ROPE, **change}
    strides = None if a.pop("strides") is None else ints(*{**ROPE, **change}["strides"])
    v = list(a.values())
    return getattr(lib, name)(*v[:9], strides, *v[9:], None)


@pytest.mark.parametrize(("change", "code", "message"), [
    (dict(q=None), "FA_ERR_NULL_POINTER", "null pointer"),
    (dict(sin=None), "FA_ERR_NULL_POINTER", "null pointer"),
    (dict(strides=None), "FA_ERR_NULL_POINTER", "null pointer"),
    (dict(q_weight=None), "FA_ERR_NULL_POINTER", "one of the two norm weights"),
    (dict(B=0), "FA_ERR_BAD_SHAPE", "must be positive"),
    (dict(P=0), "FA_ERR_BAD_SHAPE", "must be positive"),
    (dict(N=-1), "FA_ERR_BAD_SHAPE", "must be positive"),
    (dict(D=60), "FA_ERR_HEAD_DIM", "multiple of 8 up to 128"),
    (dict(D=136), "FA_ERR_HEAD_DIM", "multiple of 8 up to 128"),
    (dict(R=72), "FA_ERR_HEAD_DIM", "multiple of 16"),
    (dict(R=24), "FA_ERR_HEAD_DIM", "multiple of 16"),
    (dict(R=0), "FA_ERR_HEAD_DIM", "multiple of 16"),
    (dict(B=1 << 20, N=1 << 11), "FA_ERR_TOO_LARGE", "too many"),
    (dict(Hq=1 << 15), "FA_ERR_TOO_LARGE", "too many"),
    (dict(eps=-1.0), "FA_ERR_BAD_SCALE", "eps"),
    (dict(eps=float("inf")), "FA_ERR_BAD_SCALE", "eps"),
    (dict(flags=8), "FA_ERR_BAD_SHAPE", "flags"),
    (dict(k_out=P + 8), "FA_ERR_MISALIGNED", "16-byte"),
    (dict(cos=P + 4), "FA_ERR_MISALIGNED", "16-byte"),
    (dict(strides=(2048, 512, 60, 1024, 512, 64, 8, 1)), "FA_ERR_BAD_STRIDE", "the query"),
    (dict(strides=(2048, 512, 64, -1024, 512, 64, 8, 1)), "FA_ERR_BAD_STRIDE", "the key"),
])
@pytest.mark.parametrize("name", ["fa_qk_norm_rope", "fa_qk_norm_rope_bf16"])
def test_rope_rejects(lib, name, change, code, message):
    rejected(rope(lib, name, **change), code, message)
    assert name in _lib.last_error()


def rope_bwd(lib, ws_bytes=1 << 30, ws=P, **change):
    a = dict(gq=P, gk=P, q=P, k=P, dq=P, dk=P, dqw=P, dkw=P, cos=P, sin=P, positions=None, qw=P, kw=P,
             strides=(2048, 512, 64, 1024, 512, 64) * 2 + (0, 0), B=2, Hq=4, Hkv=2, N=8, D=64, R=64,
             P=8, eps=1e-6, flags=0)
    a.update(change)
    strides = ints(*a.pop("strides"))
    v = list(a.values())
    return lib.fa_qk_norm_rope_bwd(*v[:13], strides, *v[13:], ws, ws_bytes, None)


def test_rope_bwd_rejects(lib):
    need = lib.fa_qk_norm_rope_bwd_workspace_bytes(2, 4, 2, 8, 64)
    assert need > 0 and need % (64 * 4) == 0
    rejected(rope_bwd(lib, ws_bytes=need - 1), "FA_ERR_BAD_SHAPE", "smaller than")
    rejected(rope_bwd(lib, ws=None), "FA_ERR_NULL_POINTER", "null pointer")
    rejected(rope_bwd(lib, gk=None), "FA_ERR_NULL_POINTER", "null pointer")
    rejected(rope_bwd(lib, q=None), "FA_ERR_NULL_POINTER", "null pointer")
    rejected(rope_bwd(lib, kw=None), "FA_ERR_NULL_POINTER", "norm weights")
    rejected(rope_bwd(lib, dq=P + 2), "FA_ERR_MISALIGNED", "16-byte")
    rejected(rope_bwd(lib, strides=(2048, 512, 64, 1024, 512, 64, 2048, 512, 7, 1024, 512, 64, 0, 0)),
             "FA_ERR_BAD_STRIDE", "the query")
    rejected(lib.fa_qk_norm_rope_bwd_workspace_bytes(2, 4, 2, 8, 65), "FA_ERR_HEAD_DIM", "multiple of 8")
    rejected(lib.fa_qk_norm_rope_bwd_workspace_bytes(0, 4, 2, 8, 64), "FA_ERR_BAD_SHAPE", "positive")


@pytest.mark.parametrize(("change", "code", "message"), [
    (dict(positions=P + 2), "FA_ERR_MISALIGNED", "4-byte"),
    (dict(positions=P + 4, flags=4), "FA_ERR_MISALIGNED", "8-byte"),
    (dict(q_weight=P + 1), "FA_ERR_MISALIGNED", "2-byte"),
    (dict(k_weight=P + 1), "FA_ERR_MISALIGNED", "2-byte"),
    (dict(k_weight=P + 2, flags=2), "FA_ERR_MISALIGNED", "4-byte"),
    (dict(strides=(2048, 512, 64, 1024, 512, 64, -8, 1)), "FA_ERR_BAD_STRIDE", "the positions"),
    (dict(strides=(2048, 512, 64, 1024, 512, 64, 8, -1)), "FA_ERR_BAD_STRIDE", "the positions"),
])
def test_rope_rejects_odd_positions_and_weights(lib, change, code, message):
    for name in ("fa_qk_norm_rope", "fa_qk_norm_rope_bf16"):
        rejected(rope(lib, name, **change), code, message)
    change = {{"q_weight": "qw", "k_weight": "kw"}.get(n, n): v for n, v in change.items()}
    if "strides" in change:
        change.update(positions=P, strides=(2048, 512, 64, 1024, 512, 64) * 2 + change["strides"][6:])
    rejected(rope_bwd(lib, **change), code, message)


@pytest.mark.parametrize(("change", "message"), [
    (dict(dqw=P + 1), "2-byte"), (dict(dkw=P + 1), "2-byte"), (dict(dkw=P + 2, flags=2), "4-byte"),
])
def test_rope_bwd_rejects_odd_weight_gradients(lib, change, message):
    rejected(rope_bwd(lib, **change), "FA_ERR_MISALIGNED", message)


def plan(lib, **change):
    a = dict(table=P, table_stride=4, lengths=P, new=P, free=P, start=None, slots=P, positions=P,
             starts=P, lengths_out=P, free_out=P, B=2, M=4, S=16, F=8, T=8)
    a.update(change)
    return lib.fa_paged_plan(*a.values(), None)


@pytest.mark.parametrize(("change", "code", "message"), [
    (dict(S=0), "FA_ERR_BAD_SHAPE", "page size"),
    (dict(S=40), "FA_ERR_BAD_SHAPE", "page size"),
    (dict(M=0), "FA_ERR_BAD_SHAPE", "columns"),
    (dict(M=1 << 27), "FA_ERR_TOO_LARGE", "too many"),
    (dict(B=-1), "FA_ERR_BAD_SHAPE", "negative"),
    (dict(T=1 << 30), "FA_ERR_TOO_LARGE", "too many"),
    (dict(F=1 << 31), "FA_ERR_TOO_LARGE", "too many"),
    (dict(table=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(free=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(slots=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(starts=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(slots=P + 4), "FA_ERR_MISALIGNED", "8-byte"),
    (dict(lengths=P + 2), "FA_ERR_MISALIGNED", "4-byte"),
    (dict(table_stride=3), "FA_ERR_BAD_STRIDE", "overlap"),
])
def test_plan_rejects(lib, change, code, message):
    rejected(plan(lib, **change), code, message)


def store(lib, **change):
    a = dict(key=P, value=P, k_cache=P, v_cache=P, slots=P, strides=(128, 64, 128, 64, 2048, 1024, 64),
             T=3, H=2, D=64, pages=4, S=16)
    a.update(change)
    v = list(a.values())
    return lib.fa_paged_store(*v[:5], ints(*v[5]), *v[6:], None)


@pytest.mark.parametrize(("change", "code", "message"), [
    (dict(key=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(T=-1), "FA_ERR_BAD_SHAPE", "positive"),
    (dict(H=0), "FA_ERR_BAD_SHAPE", "positive"),
    (dict(D=4), "FA_ERR_HEAD_DIM", "multiple of 8"),
    (dict(S=8), "FA_ERR_BAD_SHAPE", "page size"),
    (dict(pages=0), "FA_ERR_BAD_SHAPE", "pages"),
    (dict(T=1 << 31), "FA_ERR_TOO_LARGE", "too many"),
    (dict(v_cache=P + 8), "FA_ERR_MISALIGNED", "16-byte"),
    (dict(strides=(128, 64, 128, 64, 2048, 1024, 56)), "FA_ERR_BAD_STRIDE", "row stride"),
    (dict(strides=(128, 64, 128, 64, 2048, 1024, 1 << 25)), "FA_ERR_BAD_STRIDE", "row stride"),
    (dict(strides=(128, 60, 128, 64, 2048, 1024, 64)), "FA_ERR_BAD_STRIDE", "the keys"),
    (dict(strides=(128, 64, 1 << 40, 64, 2048, 1024, 64)), "FA_ERR_BAD_STRIDE", "the values"),
])
def test_store_rejects(lib, change, code, message):
    rejected(store(lib, **change), code, message)


def test_store_of_no_tokens_is_no_launch(lib):
    assert store(lib, T=0, key=None) == _lib.FA_OK


def paged(lib, name="fa_paged_fwd", ws=P, ws_bytes=1 << 30, **change):
    a = dict(q=P, k=P, v=P, table=P, lengths=P, o=P, strides=(256, 64, 64, 2048, 1024, 64, 100), B=2,
             Hq=4, Hkv=2, N=1, D=64, pages=4, M=100, S=16, scale=0.125)
    a.update(change)
    v = list(a.values())
    return getattr(lib, name)(*v[:6], ints(*v[6]), *v[7:], ws, ws_bytes, None)


@pytest.mark.parametrize(("change", "code", "message"), [
    (dict(q=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(lengths=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(ws=None), "FA_ERR_NULL_POINTER", "null"),
    (dict(ws_bytes=1000), "FA_ERR_BAD_SHAPE", "smaller than"),
    (dict(Hq=3), "FA_ERR_BAD_SHAPE", "divisible"),
    (dict(N=0), "FA_ERR_BAD_SHAPE", "positive"),
    (dict(D=132), "FA_ERR_HEAD_DIM", "multiple of 8"),
    (dict(S=12), "FA_ERR_BAD_SHAPE", "page size"),
    (dict(M=0), "FA_ERR_BAD_SHAPE", "columns"),
    (dict(pages=0), "FA_ERR_BAD_SHAPE", "pages"),
    (dict(B=1 << 20, M=1 << 16), "FA_ERR_TOO_LARGE", "too many"),
    (dict(o=P + 4), "FA_ERR_MISALIGNED", "16-byte"),
    (dict(table=P + 1), "FA_ERR_MISALIGNED", "4-byte"),
    (dict(scale=0.0), "FA_ERR_BAD_SCALE", "scale"),
    (dict(scale=float("nan")), "FA_ERR_BAD_SCALE", "scale"),
    (dict(strides=(256, 64, 4, 2048, 1024, 64, 100)), "FA_ERR_BAD_STRIDE", "the query"),
    (dict(strides=(256, 64, 64, 2048, 1024, 32, 100)), "FA_ERR_BAD_STRIDE", "row stride"),
    (dict(strides=(256, 64, 64, 2048, 1024, 64, -1)), "FA_ERR_BAD_STRIDE", "page table"),
])
@pytest.mark.parametrize("name", ["fa_paged_fwd", "fa_paged_fwd_bf16"])
def test_paged_rejects(lib, name, change, code, message):
    rejected(paged(lib, name, **change), code, message)
    assert name in _lib.last_error()


def test_paged_workspace(lib):
    """None for short tables; else two partials of a row block for each work-group."""
    assert lib.fa_paged_fwd_workspace_bytes(64, 32, 8, 1, 128, 64, 16) == 0       # 1024 keys
    assert lib.fa_paged_fwd_workspace_bytes(32, 32, 8, 1, 128, 128, 16) == 0      # 2048, 256 heads
    for D, width in ((64, 64), (40, 64), (8, 32), (104, 128)):
        for N, rows in ((1, 16), (4, 16), (5, 32), (100, 32)):
            assert lib.fa_paged_fwd_workspace_bytes(4, 32, 8, N, D, 4096, 16) == \
                512 * (16 + 2 * rows * (width + 1) * 4)
    rejected(lib.fa_paged_fwd_workspace_bytes(4, 32, 7, 1, 64, 4096, 16), "FA_ERR_BAD_SHAPE", "divisible")
