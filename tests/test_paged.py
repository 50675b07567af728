"""The paged key/value cache: plan, store and attention against plain implementations (whole
numbers exactly, attention in 64 bits), the PyTorch forms on the CPU and the gfx950 kernels on
the GPU, and a decoding loop that runs them together with qk_norm_rope.

Tolerance of an attention output, element by element, with A = sum_j p_j |v_j| (p the exact
probabilities), u half a step of the type (``finfo.eps / 2``): the probabilities are rounded to
the type for the product with V, u A (fp16 below 2^-14: 2^-25 each, of a row whose largest is
at least 2^7: 2^-32 sum_j |v_j|), the output once, u |o|. In float32 the scores are sums of at
most 128 products, off by (128 + 8) 2^-24 of scale sum |q| |k|, exp2 and its argument by a few
2^-24 of |s|: a relative error of e^d - 1 in numerator and denominator, 4 d A with d the sum of
the two; the sums over n keys add n 2^-24 A at most."""

from __future__ import annotations

import math
import random

import pytest
import torch

from triton_flash_attention import (_native, paged_attention, paged_cache_plan, paged_cache_store,
                                    qk_norm_rope, scaled_dot_product_attention)

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
F32 = 2.0 ** -24


def cdiv(a, b):
    return -(-a // b)


# ---- plan -------------------------------------------------------------------------------


def plan_reference(table, lengths, new, free, start, S, T):
    """The plan by a walk over the tokens: (table, slots, positions, starts, lengths, start)."""
    table = [row[:] for row in table]
    M = len(table[0]) if table else 1
    slots, positions, starts = [], [], [0]
    for b, (n, k) in enumerate(zip(lengths, new)):
        n, k = max(n, 0), max(k, 0)
        row = dict(enumerate(table[b]))  # the sequence's pages
        for j in range(cdiv(n, S), min(cdiv(n + k, S), M)):
            row[j] = free[start] if 0 <= start < len(free) else -1
            if starts[-1] + j * S - n < T:  # written by the page's first token
                table[b][j] = row[j]
            start += 1
        for p in range(n, n + k):
            page = row.get(p // S, -1)
            slots.append(page * S + p % S if page >= 0 else -1)
            positions.append(p)
        starts.append(len(slots))
    pad = T - len(slots)
    return (table, (slots + [-1] * pad)[:T], (positions + [0] * pad)[:T], starts,
            [max(n, 0) + max(k, 0) for n, k in zip(lengths, new)], max(start, 0))


def check_plan(lengths, new, S, *, M=None, free=None, start=None, T=None, seed=0, device="cpu",
               backend="torch", pad_columns=0):
    rng = random.Random(seed)
    held = [cdiv(max(n, 0), S) for n in lengths]
    width = max([1] + [cdiv(max(n, 0) + max(k, 0), S) for n, k in zip(lengths, new)])
    M = M or width
    total = sum(held) + sum(cdiv(max(n, 0) + max(k, 0), S) - h for n, k, h in zip(lengths, new, held))
    pages = list(range(total + 5))
    rng.shuffle(pages)
    table = [[pages.pop() if j < h else -7 for j in range(M)] for h in held]
    free = pages if free is None else free(pages)
    T = sum(max(k, 0) for k in new) + 3 if T is None else T
    want = plan_reference(table, lengths, new, free, start or 0, S, T)

    def ints(v, dtype=torch.int32):
        return torch.tensor(v, dtype=dtype, device=device)

    t = torch.full((len(lengths), M + pad_columns), -9, dtype=torch.int32, device=device)[:, :M]
    if lengths:
        t.copy_(ints(table))
    plan = paged_cache_plan(t, ints(lengths), ints(new), ints(free), page_size=S, num_tokens=T,
                            free_start=None if start is None else ints([start]), backend=backend)
    assert t.tolist() == want[0]
    assert plan.slots.dtype == torch.int64 and plan.slots.tolist() == want[1]
    assert plan.positions.dtype == torch.int32 and plan.positions.tolist() == want[2]
    assert plan.starts.tolist() == want[3] and plan.lengths.tolist() == want[4]
    assert plan.free_start.tolist() == [want[5]]


def ragged(n, hi, seed, lo=0):
    rng = random.Random(seed)
    return [rng.choice([lo, hi, rng.randint(lo, hi), rng.randint(lo, max(lo, hi // 8))])
            for _ in range(n)]


PLANS = [
    dict(lengths=[0], new=[1], S=16),
    dict(lengths=[15, 16, 17, 0], new=[1, 1, 1, 1], S=16),
    dict(lengths=[0, 0, 0], new=[0, 0, 0], S=16),
    dict(lengths=[], new=[], S=16),
    dict(lengths=[], new=[], S=16, T=0),
    dict(lengths=[5, 0, 47, 100], new=[0, 31, 0, 200], S=48),
    dict(lengths=ragged(37, 300, 1), new=ragged(37, 70, 2), S=16, start=2),
    dict(lengths=[3, -4, 7], new=[2, 5, -1], S=16),
    # the free pages run out; a start outside the list
    dict(lengths=[0, 10, 0], new=[40, 40, 40], S=16, free=lambda p: p[:4]),
    dict(lengths=[0, 10], new=[40, 1], S=16, free=lambda p: []),
    dict(lengths=[0, 10], new=[40, 7], S=16, start=1000),
    dict(lengths=[0, 10], new=[40, 7], S=16, start=-2),
    # more tokens than the table's row holds, than the step has rows
    dict(lengths=[30, 100, 5], new=[20, 3, 5], S=16, M=2),
    dict(lengths=[0, 3, 20], new=[50, 50, 50], S=16, T=60),
    dict(lengths=[0, 3, 20], new=[50, 50, 50], S=16, T=0),
]


@pytest.mark.parametrize("case", PLANS)
def test_plan_torch_form(case):
    check_plan(**case)


@pytest.mark.gpu
@pytest.mark.parametrize("case", PLANS)
def test_plan_kernel(case):
    check_plan(**case, device="cuda", backend="triton")


@pytest.mark.gpu
@pytest.mark.parametrize("case", [
    dict(lengths=ragged(1024, 50, 3), new=ragged(1024, 3, 4), S=16, pad_columns=3),
    dict(lengths=ragged(1025, 50, 3), new=ragged(1025, 9, 4), S=16),
    dict(lengths=ragged(5000, 20, 5), new=ragged(5000, 2, 6), S=32, start=1),
    dict(lengths=ragged(7, 4000, 7), new=ragged(7, 9000, 8), S=128),
    dict(lengths=[0] * 3000 + [7], new=[0] * 3000 + [2500], S=16),
    dict(lengths=[100000], new=[70001], S=64),
    dict(lengths=ragged(1500, 500, 9), new=ragged(1500, 700, 10), S=16),  # 300 thousand tokens
])
def test_plan_kernel_over_groups_and_blocks(case):
    check_plan(**case, device="cuda", backend="triton")


def check_plan_of_counts_past_32_bits(big, T, device, backend):
    """``big`` counts of 2^30 - 1 in the first 1024 sequences, then many of one token: the
    step's T tokens all belong to sequence 0, and only their pages are written."""
    S, M, B, most = 16, 4, 2100, (1 << 30) - 1
    i32 = dict(dtype=torch.int32, device=device)
    new = torch.ones(B, **i32)
    new[:1024] = 0
    new[:big] = most
    free = torch.arange(10, 10 + 4 * B, **i32)
    table = torch.full((B, M), -9, **i32)
    plan = paged_cache_plan(table, torch.zeros(B, **i32), new, free, page_size=S, num_tokens=T,
                            backend=backend)
    entries = torch.full((B, M), -9, dtype=torch.int32)
    entries[0, :cdiv(T, S)] = torch.arange(10, 10 + cdiv(T, S))
    assert torch.equal(table.cpu(), entries)
    t = torch.arange(T)
    assert torch.equal(plan.slots.cpu(), 10 * S + t) and torch.equal(plan.positions.cpu(), t.int())
    total = [0]
    for n in new.tolist():
        total.append(min(total[-1] + n, 1 << 62))
    assert plan.starts.tolist() == [min(n, (1 << 31) - 1) for n in total]
    assert torch.equal(plan.lengths, new) and plan.free_start.tolist() == [M * big + B - 1024]


COUNTS_PAST_32_BITS = [(2, 64), (3, 64), (4, 0), (4, 50), (4, 64), (5, 64), (8, 64), (12, 64)]


@pytest.mark.parametrize(("big", "T"), COUNTS_PAST_32_BITS)
def test_plan_torch_form_of_counts_past_32_bits(big, T):
    check_plan_of_counts_past_32_bits(big, T, "cpu", "torch")


@pytest.mark.gpu
@pytest.mark.parametrize(("big", "T"), COUNTS_PAST_32_BITS)
def test_plan_kernel_of_counts_past_32_bits(big, T):
    check_plan_of_counts_past_32_bits(big, T, "cuda", "triton")


def _plan_args():
    i = torch.int32
    return dict(page_table=torch.zeros(2, 4, dtype=i), lengths=torch.zeros(2, dtype=i),
                new_tokens=torch.ones(2, dtype=i), free_pages=torch.arange(8, dtype=i),
                page_size=16, num_tokens=2)


@pytest.mark.parametrize(("change", "error", "message"), [
    (dict(backend="x"), ValueError, "backend"),
    (dict(page_table=torch.zeros(2, 4)), ValueError, "page_table must be int32"),
    (dict(page_table=torch.zeros(8, dtype=torch.int32)), ValueError, "page_table must have shape"),
    (dict(page_table=torch.zeros(2, 0, dtype=torch.int32)), ValueError, "one column"),
    (dict(page_table=torch.zeros(1, 4, dtype=torch.int32).expand(2, 4)), ValueError, "overlap"),
    (dict(page_size=8), ValueError, "multiple of 16"),
    (dict(page_size=24), ValueError, "multiple of 16"),
    (dict(page_size=0), ValueError, "multiple of 16"),
    (dict(page_size=True), ValueError, "multiple of 16"),
    (dict(page_size=1 << 29), ValueError, "more than"),
    (dict(lengths=torch.zeros(2, dtype=torch.int64)), ValueError, "lengths must be int32"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), ValueError, "lengths must have shape"),
    (dict(new_tokens=[1, 1]), TypeError, "new_tokens"),
    (dict(free_pages=torch.zeros(2, 2, dtype=torch.int32)), ValueError, "free_pages"),
    (dict(free_start=torch.zeros(2, dtype=torch.int32)), ValueError, "free_start"),
    (dict(free_start=3), TypeError, "free_start"),
    (dict(num_tokens=-1), ValueError, "num_tokens"),
    (dict(num_tokens=2.0), ValueError, "num_tokens"),
    (dict(backend="triton"), RuntimeError, "CUDA tensor"),
])
def test_plan_refusals(change, error, message):
    with pytest.raises(error, match=message):
        paged_cache_plan(**{**_plan_args(), **change})


# ---- store ------------------------------------------------------------------------------


def check_store(T, H, D, S, dtype, *, layout="heads", cache_layout="heads", device="cpu",
                backend="torch", pages=None, seed=0):
    gen = torch.Generator().manual_seed(seed)
    pages = pages or cdiv(T, S) + 2
    if layout == "fused":
        f = torch.randn(T, 4 * H, D, generator=gen).to(dtype).to(device)
        key, value = f[:, 2 * H:3 * H], f[:, 3 * H:]
    else:
        key, value = (torch.randn(T, H, D, generator=gen).to(dtype).to(device) for _ in range(2))
    shape = (pages, S, H, D) if cache_layout == "tokens" else (pages, H, S, D)
    caches = [torch.randn(shape, generator=gen).to(dtype).to(device) for _ in range(2)]
    views = [c.transpose(1, 2) if cache_layout == "tokens" else c for c in caches]
    slots = torch.randperm(pages * S, generator=gen)[:T]
    outside = [-1, -5, pages * S, 1 << 40, -(1 << 50)]
    for i in range(0, T, 3):
        slots[i] = outside[i // 3 % len(outside)]
    want = [v.clone() for v in views]
    for w, t in zip(want, (key, value)):
        for i, s in enumerate(slots.tolist()):
            if 0 <= s < pages * S:
                w[s // S, :, s % S] = t[i]
    version = views[0]._version
    paged_cache_store(key, value, *views, slots.to(device), backend=backend)
    assert all(torch.equal(a, b) for a, b in zip(views, want))
    assert T == 0 or views[0]._version > version


STORES = [
    (1, 1, 8, 16, "heads", "heads"),
    (0, 2, 64, 16, "heads", "heads"),
    (7, 2, 64, 16, "fused", "tokens"),
    (33, 3, 40, 48, "heads", "tokens"),
    (50, 8, 128, 32, "fused", "heads"),
]


@pytest.mark.parametrize("case", STORES)
def test_store_torch_form(case):
    T, H, D, S, layout, cache = case
    check_store(T, H, D, S, torch.bfloat16, layout=layout, cache_layout=cache)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", STORES + [(300, 16, 96, 16, "fused", "heads"),
                                           (1000, 1, 32, 64, "heads", "heads"),
                                           (515, 5, 128, 16, "heads", "tokens")])
def test_store_kernel(case, dtype):
    T, H, D, S, layout, cache = case
    check_store(T, H, D, S, dtype, layout=layout, cache_layout=cache, device="cuda",
                backend="triton", seed=T)


@pytest.mark.gpu
def test_store_kernel_copies_keys_it_cannot_read():
    gen = torch.Generator().manual_seed(1)
    wide = torch.randn(5, 2, 33, generator=gen).half().cuda()
    key, value = wide[..., 1:], wide[..., :32]
    caches = [torch.zeros(2, 2, 16, 32, dtype=torch.float16, device="cuda") for _ in range(2)]
    slots = torch.tensor([0, 31, 5, -1, 7], device="cuda")
    paged_cache_store(key, value, *caches, slots, backend="triton")
    for c, t in zip(caches, (key, value)):
        assert torch.equal(c[1, :, 15], t[1]) and torch.equal(c[0, :, 5], t[2])


@pytest.mark.gpu
def test_store_kernel_of_more_tokens_than_a_grid_holds():
    """2^24 blocks of two tokens and some: rows 16 bytes apart of one buffer, a few with slots."""
    T, H, D, S = (1 << 25) + 5, 8, 128, 16
    base = torch.empty(8 * T + 9 * 1024, dtype=torch.float16, device="cuda").normal_()
    key, value = (t.as_strided((T, H, D), (8, 1024, 1)) for t in (base, base[1024:]))
    edge = (1 << 25) - 2
    chosen = torch.tensor([0, 1, 77, edge - 1, edge, edge + 1, 1 << 25, T - 2, T - 1], device="cuda")
    slots = torch.full((T,), -1, dtype=torch.int64, device="cuda")
    slots[chosen] = torch.arange(9, device="cuda") * 5
    caches = [torch.zeros(3, H, S, D, dtype=torch.float16, device="cuda") for _ in range(2)]
    paged_cache_store(key, value, *caches, slots, backend="triton")
    for c, t in zip(caches, (key, value)):
        rows = c.transpose(1, 2).reshape(3 * S, H, D)
        assert torch.equal(rows[:45:5], t[chosen])
        rows[:45:5] = 0
        assert not rows.any()


_SAME = torch.zeros(4, 2, 16, 32).half()


def _store_args(device="cpu", dtype=torch.float16):
    z = dict(dtype=dtype, device=device)
    return dict(key=torch.zeros(3, 2, 32, **z), value=torch.zeros(3, 2, 32, **z),
                key_cache=torch.zeros(4, 2, 16, 32, **z), value_cache=torch.zeros(4, 2, 16, 32, **z),
                slots=torch.arange(3, device=device))


@pytest.mark.parametrize(("change", "error", "message"), [
    (dict(backend="x"), ValueError, "backend"),
    (dict(key=torch.zeros(3, 2, 16).half()), ValueError, "same shape"),
    (dict(key=torch.zeros(3, 64).half()), ValueError, "key must have shape"),
    (dict(key=torch.zeros(3, 1, 32).half(), value=torch.zeros(3, 1, 32).half()), ValueError,
     "key and value must have shape"),
    (dict(key_cache=torch.zeros(4, 2, 24, 32).half(), value_cache=torch.zeros(4, 2, 24, 32).half()),
     ValueError, "multiple of 16"),
    (dict(value_cache=torch.zeros(5, 2, 16, 32).half()), ValueError, "same shape"),
    (dict(value_cache=torch.zeros(4, 2, 16, 32)), ValueError, "share a device and a dtype"),
    (dict(key=torch.zeros(3, 2, 32)), ValueError, "same dtype"),
    (dict(slots=torch.zeros(4).long()), ValueError, "slots must have shape"),
    (dict(slots=torch.zeros(3).int()), ValueError, "int64"),
    (dict(slots=[0, 1, 2]), TypeError, "slots"),
    (dict(key=torch.zeros(3, 2, 32).half().requires_grad_()), RuntimeError, "no gradients"),
    (dict(key_cache=torch.zeros(1, 2, 16, 32).half().expand(4, 2, 16, 32)), ValueError, "expanded"),
    (dict(key_cache=_SAME, value_cache=_SAME), ValueError, "different tensors"),
    (dict(backend="triton"), RuntimeError, "CUDA tensor"),
])
def test_store_refusals(change, error, message):
    with pytest.raises(error, match=message):
        paged_cache_store(**{**_store_args(), **change})


@pytest.mark.gpu
def test_store_kernel_refuses_caches_it_cannot_address():
    a = _store_args("cuda")
    with pytest.raises(RuntimeError, match="same strides"):
        paged_cache_store(**{**a, "key_cache": torch.zeros(4, 16, 2, 32, device="cuda").half()
                             .transpose(1, 2)}, backend="triton")
    odd, odd2 = (torch.zeros(4, 2, 16, 33, device="cuda").half()[..., 1:] for _ in range(2))
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        paged_cache_store(**{**a, "key_cache": odd, "value_cache": odd2}, backend="triton")
    b = _store_args("cuda", torch.float32)
    with pytest.raises(RuntimeError, match="float16 and bfloat16"):
        paged_cache_store(**b, backend="triton")


# ---- attention --------------------------------------------------------------------------


def make_paged(lengths, Hkv, S, D, dtype, *, seed=0, layout="heads", M=None, fill=math.nan,
               device="cpu", spare=3, scale=1.0):
    """A cache that holds ``fill`` wherever no token lies, its table, and the dense keys and
    values [n, Hkv, D] of each sequence (float64)."""
    gen = torch.Generator().manual_seed(seed)
    held = [cdiv(n, S) for n in lengths]
    M = M or max(1, *held)
    pages = sum(held) + spare
    order = torch.randperm(pages, generator=gen).tolist()
    shape = (pages, S, Hkv, D) if layout == "tokens" else (pages, Hkv, S, D)
    caches = [torch.full(shape, fill).to(dtype) for _ in range(2)]
    views = [c.transpose(1, 2) if layout == "tokens" else c for c in caches]
    table, dense = torch.full((len(lengths), M), -1, dtype=torch.int32), []
    for b, n in enumerate(lengths):
        kv = [(torch.randn(n, Hkv, D, generator=gen) * scale).to(dtype) for _ in range(2)]
        for j in range(held[b]):
            page = order.pop()
            table[b, j] = page
            for c, t in zip(views, kv):
                part = t[j * S:(j + 1) * S]
                c[page, :, :part.shape[0]] = part.transpose(0, 1)
        dense.append([t.double() for t in kv])
    caches = [c.to(device) for c in caches]
    views = [c.transpose(1, 2) if layout == "tokens" else c for c in caches]
    return views, table.to(device), torch.tensor(lengths, dtype=torch.int32, device=device), dense


def attention_reference(q, dense, scale, dtype):
    """(o, its bound) [B, Hq, N, D] in float64."""
    q = q.double().cpu()
    B, Hq, N, D = q.shape
    o, bound = torch.zeros_like(q), torch.zeros_like(q)
    for b, (k, v) in enumerate(dense):
        n, H = k.shape[:2]
        for i in range(N):
            seen = n - N + i + 1
            if seen <= 0:
                continue
            kk, vv = (t[:seen].repeat_interleave(Hq // H, 1).transpose(0, 1) for t in (k, v))
            qi = q[b, :, i, :, None]
            s = (kk @ qi).squeeze(-1) * scale
            p = torch.softmax(s, -1)[:, None]
            o[b, :, i] = (p @ vv).squeeze(1)
            A = (p @ vv.abs()).squeeze(1)
            size = (kk.abs() @ qi.abs()).squeeze(-1).amax(-1) * abs(scale)
            d = (136 * size + 8 * s.abs().amax(-1)) * F32
            bound[b, :, i] = (A * (HALF[dtype] + seen * F32 + 4 * d[:, None])
                              + (2.0 ** -32 * vv.abs().sum(1) if dtype == torch.float16 else 0))
    return o, bound


def check_attend(lengths, Hq, Hkv, N, D, S, dtype, *, layout="heads", scale=None, seed=0,
                 device="cpu", backend="torch", q_layout="heads", spread=1.0, **cache):
    views, table, lens, dense = make_paged(lengths, Hkv, S, D, dtype, seed=seed, layout=layout,
                                           device=device, **cache)
    gen = torch.Generator().manual_seed(seed + 1)
    B = len(lengths)
    if q_layout == "tokens":
        q = (torch.randn(B, N, Hq + 3, D, generator=gen) * spread).to(dtype).to(device)
        q = q[:, :, 1:Hq + 1].transpose(1, 2)
    else:
        q = (torch.randn(B, Hq, N, D, generator=gen) * spread).to(dtype).to(device)
    o = paged_attention(q, *views, table, lens, scale=scale, enable_gqa=Hq != Hkv, backend=backend)
    want, bound = attention_reference(q, dense, D ** -0.5 if scale is None else scale, dtype)
    assert o.shape == want.shape and o.is_contiguous() and o.dtype == dtype
    off = (o.double().cpu() - want).abs()
    limit = HALF[dtype] * want.abs() * 1.01 + bound * 1.01 + 2.0 ** -24
    assert bool((off <= limit).all()), f"{(off / limit).max().item():.3f} of the bound"
    return o


ATTENDS = [
    # lengths, Hq, Hkv, N, D, S
    ([1], 1, 1, 1, 32, 16),
    ([0, 1, 2, 15], 4, 2, 1, 64, 16),
    ([16, 17, 31, 32, 33, 0], 8, 2, 1, 128, 16),
    ([5, 0, 70], 6, 2, 4, 64, 32),            # some queries see no key
    ([100, 3, 47, 48, 49], 4, 4, 1, 40, 48),
    ([129, 64], 16, 1, 1, 128, 64),
    ([33, 90], 12, 2, 3, 80, 16),             # 18 rows a head: two row blocks
    ([200], 8, 1, 5, 32, 128),                # 40 rows: three
]


@pytest.mark.parametrize("case", ATTENDS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_attention_torch_form(case, dtype):
    check_attend(*case, dtype)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.7])
def test_attention_torch_form_scales(scale):
    check_attend([40, 7], 4, 2, 2, 32, 16, torch.float32, scale=scale)


def test_attention_torch_form_has_gradients():
    views, table, lens, _ = make_paged([5, 0, 20], 1, 16, 8, torch.float64, fill=0.0)
    leaves = [torch.randn(3, 2, 2, 8, dtype=torch.float64, requires_grad=True),
              *(v.clone().requires_grad_() for v in views)]
    assert torch.autograd.gradcheck(
        lambda q, k, v: paged_attention(q, k, v, table, lens, enable_gqa=True), leaves,
        fast_mode=True)


def bad_rows(device, backend, dtype):
    """Lengths and pages that do not exist make their own sequence NaN and no other."""
    views, table, lens, dense = make_paged([40, 40, 40, 40, 40, 40], 2, 16, 64, dtype, M=4,
                                           fill=0.0, device=device)
    q = torch.randn(6, 4, 1, 64).to(dtype).to(device)
    pages = views[0].shape[0]
    lens[1], lens[2] = -1, 65
    table[3, 1], table[4, 2] = pages, -2
    table[5, 3] = 1 << 30  # behind the length: not looked at
    o = paged_attention(q, *views, table, lens, enable_gqa=True, backend=backend).cpu()
    want, _ = attention_reference(q, dense, 0.125, dtype)
    for b in range(6):
        if b in (1, 2, 3, 4):
            assert o[b].isnan().all(), b
        else:
            assert torch.allclose(o[b].double(), want[b], atol=2e-2), b


def test_attention_torch_form_bad_rows():
    bad_rows("cpu", "torch", torch.float32)


def _attend_args(device="cpu", dtype=torch.float16):
    z = dict(dtype=dtype, device=device)
    i = dict(dtype=torch.int32, device=device)
    return dict(query=torch.zeros(2, 4, 1, 32, **z), key_cache=torch.zeros(4, 2, 16, 32, **z),
                value_cache=torch.zeros(4, 2, 16, 32, **z), page_table=torch.zeros(2, 3, **i),
                lengths=torch.ones(2, **i), enable_gqa=True)


@pytest.mark.parametrize(("change", "error", "message"), [
    (dict(backend="x"), ValueError, "backend"),
    (dict(enable_gqa=1), TypeError, "enable_gqa"),
    (dict(enable_gqa=False), ValueError, "enable_gqa=True"),
    (dict(scale=float("inf")), ValueError, "scale"),
    (dict(query=torch.zeros(2, 4, 32).half()), ValueError, "query must have shape"),
    (dict(query=torch.zeros(2, 4, 0, 32).half()), ValueError, "greater than zero"),
    (dict(query=torch.zeros(2, 4, 1, 32)), ValueError, "same dtype"),
    (dict(query=torch.zeros(2, 4, 1, 64).half()), ValueError, "head dimensions"),
    (dict(query=torch.zeros(2, 3, 1, 32).half()), ValueError, "divisible"),
    (dict(query=torch.zeros(3, 4, 1, 32).half()), ValueError, "a row for each sequence"),
    (dict(page_table=torch.zeros(2, 3)), ValueError, "page_table must be int32"),
    (dict(lengths=torch.ones(2).long()), ValueError, "lengths must be int32"),
    (dict(lengths=torch.ones(2, 1).int()), ValueError, "lengths must have shape"),
    (dict(key_cache=torch.zeros(4, 2, 20, 32).half(), value_cache=torch.zeros(4, 2, 20, 32).half()),
     ValueError, "multiple of 16"),
    (dict(value_cache=torch.zeros(4, 2, 16, 32)), ValueError, "share a device and a dtype"),
    (dict(backend="triton"), RuntimeError, "CUDA tensor"),
])
def test_attention_refusals(change, error, message):
    with pytest.raises(error, match=message):
        paged_attention(**{**_attend_args(), **change})


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
@pytest.mark.parametrize("case", ATTENDS)
def test_attention_kernel(case, layout, dtype):
    check_attend(*case, dtype, layout=layout, q_layout=layout, device="cuda", backend="triton")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", [
    ([3001], 32, 8, 1, 128, 16),              # one sequence over the whole chip
    ([9000, 1, 130], 8, 1, 1, 64, 64),        # more than 32 units a wave
    (ragged(40, 900, 9), 8, 8, 1, 64, 16),
    (ragged(300, 90, 10, 1), 4, 2, 2, 32, 32),
    (ragged(9, 2500, 11), 16, 2, 5, 96, 16),
    ([2049, 2048, 4000], 4, 4, 4, 128, 48),
    ([20000], 2, 1, 17, 32, 16),              # 34 rows
])
def test_attention_kernel_over_work_groups(case, dtype):
    o = check_attend(*case, dtype, device="cuda", backend="triton", M=cdiv(max(case[0]), case[5]) + 3)
    again = check_attend(*case, dtype, device="cuda", backend="triton",
                         M=cdiv(max(case[0]), case[5]) + 3)
    assert torch.equal(o, again)


@pytest.mark.gpu
@pytest.mark.parametrize("case", [
    # tables wide enough for the launch that splits, filled a little or a lot
    ([40], 4, 1, 1, 64, 16, 80),              # lines with room for every head: one round
    ([40, 300, 7, 0, 1], 8, 2, 1, 128, 16, 80),
    ([2000, 3, 2000], 8, 8, 1, 64, 16, 130),  # two rounds
    ([0, 0, 0], 4, 2, 1, 32, 16, 100),
    (ragged(600, 30, 12), 2, 2, 1, 32, 16, 70),    # several sequences a thread
    (ragged(1100, 9, 13), 4, 4, 1, 64, 16, 70),    # many short pieces a work-group
    (ragged(24, 1100, 14), 16, 4, 3, 128, 16, 90),
    ([17] * 40 + [5000] + [17] * 40, 8, 2, 1, 64, 16, 320),
    ([1500] * 64, 4, 4, 1, 32, 16, 100),      # 256 heads, at most 2048 keys: one launch
])
def test_attention_kernel_in_wide_tables(case):
    *shape, M = case
    check_attend(*shape, torch.float16, M=M, device="cuda", backend="triton")


@pytest.mark.gpu
@pytest.mark.parametrize("case", [
    # heads that share a line, token by token: consecutive stretches an XCD
    (ragged(24, 1500, 15), 8, 4, 1, 32, 16, 100),
    ([9000, 1, 130], 4, 2, 5, 24, 16, 600),
    (ragged(40, 900, 16), 3, 3, 1, 56, 32, 70),
    ([1200, 5], 2, 2, 1, 8, 16, 80),          # fewer work-groups than the chip holds
])
def test_attention_kernel_of_heads_that_share_lines(case):
    *shape, M = case
    o = check_attend(*shape, torch.float16, M=M, layout="tokens", device="cuda", backend="triton")
    assert torch.equal(o, check_attend(*shape, torch.float16, M=M, device="cuda", backend="triton"))


@pytest.mark.gpu
def test_plan_kernel_reads_strided_lengths():
    lengths, new = (torch.tensor(v, dtype=torch.int32, device="cuda").view(4, 2)[:, 0]
                    for v in ([3, 9, 20, 9, 0, 9, 33, 9], [1, 7, 2, 7, 5, 7, 0, 7]))
    free = torch.arange(20, dtype=torch.int32, device="cuda")[::2]
    tables = [torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4).t().contiguous()
              .repeat(1, 2) for _ in range(2)]
    start = torch.tensor(2, dtype=torch.int32, device="cuda")
    plans = [paged_cache_plan(t, lengths, new, free, page_size=16, num_tokens=9, free_start=start,
                              backend=b) for t, b in zip(tables, ("triton", "torch"))]
    assert torch.equal(*tables)
    assert all(torch.equal(a, b) for a, b in zip(*plans))


@pytest.mark.gpu
def test_attention_kernel_reads_a_transposed_table():
    views, table, lens, dense = make_paged([100, 37], 2, 16, 32, torch.float16, device="cuda")
    q = torch.randn(2, 4, 1, 32).half().cuda()
    want = paged_attention(q, *views, table, lens, enable_gqa=True, backend="triton")
    odd = table.t().contiguous().t()
    assert odd.stride(1) != 1
    strided = torch.stack([lens, lens * 0], 1)[:, 0]
    got = paged_attention(q, *views, odd, strided, enable_gqa=True, backend="triton")
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_attention_kernel_many_units_a_wave():
    """Stretches of hundreds of units: each wave takes new pages many times."""
    lengths = [32768 - 1777 * b for b in range(16)]
    check_attend(lengths, 16, 16, 1, 8, 128, torch.float16, device="cuda", backend="triton")


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(16))
def test_attention_kernel_random(seed):
    rng = random.Random(seed)
    Hkv = rng.choice([1, 2, 3, 5])
    S, B = rng.choice([16, 32, 48, 80]), rng.choice([1, 2, 7, 33, 90])
    hi = rng.choice([60, 700, 3000]) if B < 90 else 300
    lengths = ragged(B, hi, seed)
    check_attend(lengths, Hkv * rng.choice([1, 2, 4, 6]), Hkv, rng.choice([1, 1, 2, 3]),
                 rng.choice([8, 32, 48, 64, 104, 128]), S, rng.choice([torch.float16, torch.bfloat16]),
                 layout=rng.choice(["heads", "tokens"]), q_layout=rng.choice(["heads", "tokens"]),
                 M=max(cdiv(hi, S), rng.choice([1, cdiv(1100, S), cdiv(9000, S)])), seed=seed,
                 device="cuda", backend="triton")


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.3, 1.7, 1e-40])
def test_attention_kernel_scales(scale):
    check_attend([400, 7, 0], 4, 2, 2, 64, 16, torch.float16, scale=scale, device="cuda",
                 backend="triton")


@pytest.mark.gpu
def test_attention_kernel_large_scores():
    """Scores in the thousands: one key takes all the weight, wherever it lies."""
    check_attend([777, 2000], 8, 2, 1, 64, 16, torch.bfloat16, spread=30.0, device="cuda",
                 backend="triton")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize(("B", "n"), [(1, 896), (512, 32768)])
def test_attention_kernel_counts_the_many_small_weights_of_long_rows(B, n, dtype):
    """Every wave's first unit holds the largest score, 18 above all others: 2^-26 of its weight
    each, and the only ones with a value. All sequences share the pages."""
    S, D = 16, 32
    k, v = (torch.zeros(2, 1, S, D, dtype=dtype, device="cuda") for _ in range(2))
    k[1, 0, 0, 0], v[:] = 18.0, 1.0
    v[1, 0, 0] = 0.0
    table = torch.zeros(1, n // S, dtype=torch.int32, device="cuda")
    table[0, :8:2] = 1
    q = torch.zeros(B, 1, 1, D, dtype=dtype, device="cuda")
    q[..., 0] = 1.0
    o = paged_attention(q, k, v, table.expand(B, -1),
                        torch.full((B,), n, dtype=torch.int32, device="cuda"), scale=1.0,
                        backend="triton").double().cpu()
    peaks, small = 4, (n - 4) * math.exp(-18.0)
    want = small / (peaks + small)
    d = (136 + 8) * 18 * F32
    bound = want * (2 * HALF[dtype] + n * F32 + 4 * d) + (
        n / peaks * 2.0 ** -32 + 2.0 ** -25 if dtype == torch.float16 else 0)
    assert float((o - want).abs().max()) <= bound


def large_values(kind, lengths, M, dtype, device, backend):
    """Values of up to 2^127, whose sums have no room in float32, under scores that are random,
    all equal, or grow with the key: the output is no larger than the largest value."""
    S, D, Hq, Hkv, N = 16, 32, 4, 2, 2
    views, table, lens, dense = make_paged(lengths, Hkv, S, D, dtype, M=M, seed=6)
    views[1].abs_().mul_(2.0 ** 124)  # exact
    for b, (k, v) in enumerate(dense):
        v.abs_().mul_(2.0 ** 124)
        at = torch.arange(lengths[b])
        if kind == "equal":
            k.zero_()
        elif kind == "grow":  # by steps of 4: a weight of e^4 against the keys before
            k.zero_()[:, :, 0] = (at // 40 * 4.0).clamp(max=120.0)[:, None]
        views[0][table[b].long()[at // S], :, at % S] = k.to(dtype)
    q = torch.randn(len(lengths), Hq, N, D, generator=torch.Generator().manual_seed(7)).to(dtype)
    if kind == "grow":
        q[..., 0] = 1.0
    views = [v.to(device) for v in views]
    o = paged_attention(q.to(device), *views, table.to(device), lens.to(device), scale=1.0,
                        enable_gqa=True, backend=backend)
    want, bound = attention_reference(q, dense, 1.0, dtype)
    limit = HALF[dtype] * want.abs() * 1.01 + bound * 1.01
    assert bool(((o.double().cpu() - want).abs() <= limit).all())


LARGE_VALUES = [(kind, *c) for kind in ("random", "equal", "grow")
                for c in (([300, 1, 33], None), ([9000, 40, 1200], 600))]


@pytest.mark.parametrize(("kind", "lengths", "M"), LARGE_VALUES)
def test_attention_torch_form_large_values(kind, lengths, M):
    large_values(kind, lengths, M, torch.bfloat16, "cpu", "torch")


@pytest.mark.gpu
@pytest.mark.parametrize(("kind", "lengths", "M"), LARGE_VALUES)
def test_attention_kernel_large_values(kind, lengths, M):
    large_values(kind, lengths, M, torch.bfloat16, "cuda", "triton")


@pytest.mark.gpu
@pytest.mark.parametrize("fill", [math.inf, -math.inf, 65504.0])
def test_attention_kernel_never_sees_what_lies_behind_the_length(fill):
    check_attend([1, 33, 300, 0], 8, 2, 1, 128, 32, torch.float16, fill=fill, device="cuda",
                 backend="triton")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_kernel_bad_rows(dtype):
    bad_rows("cuda", "triton", dtype)


@pytest.mark.gpu
def test_kernels_take_any_stride_of_one_element_dimensions():
    """One page, one head: the strides of such dimensions say nothing."""
    gen = torch.Generator().manual_seed(5)
    kc = torch.randn(16, 64, generator=gen).half().cuda().as_strided((1, 1, 16, 64), (3, 5, 64, 1))
    vc = torch.randn(16, 64, generator=gen).half().cuda().as_strided((1, 1, 16, 64), (7, 0, 64, 1))
    key, value = (torch.randn(2, 1, 64, generator=gen).half().cuda() for _ in range(2))
    paged_cache_store(key, value, kc, vc, torch.tensor([3, 0]).cuda(), backend="triton")
    assert torch.equal(kc[0, 0, 3], key[0, 0]) and torch.equal(vc[0, 0, 0], value[1, 0])
    q = torch.randn(1, 4, 1, 64, generator=gen).half().cuda()
    o = paged_attention(q, kc, vc, torch.zeros(1, 1, dtype=torch.int32).cuda(),
                        torch.tensor([11], dtype=torch.int32).cuda(), enable_gqa=True,
                        backend="triton")
    dense = [[t[0, :, :11].transpose(0, 1).double().cpu() for t in (kc, vc)]]
    want, bound = attention_reference(q, dense, 0.125, torch.float16)
    assert ((o.double().cpu() - want).abs() <= HALF[torch.float16] * want.abs() * 1.01 + bound).all()


@pytest.mark.gpu
def test_attention_kernel_bad_page_of_a_long_sequence():
    """One bad page among many work-groups' pieces."""
    views, table, lens, _ = make_paged([5000, 64], 1, 16, 64, torch.float16, device="cuda", fill=0.0)
    q = torch.randn(2, 4, 1, 64).half().cuda()
    good = paged_attention(q, *views, table, lens, enable_gqa=True, backend="triton")
    for j in (0, 100, 312):
        t = table.clone()
        t[0, j] = -1
        o = paged_attention(q, *views, t, lens, enable_gqa=True, backend="triton")
        assert o[0].isnan().all() and torch.equal(o[1], good[1])


@pytest.mark.gpu
def test_attention_kernel_matches_the_dense_call():
    views, table, lens, dense = make_paged([513] * 3, 2, 16, 64, torch.float16, device="cuda")
    q = torch.randn(3, 8, 1, 64).half().cuda()
    o = paged_attention(q, *views, table, lens, enable_gqa=True, backend="triton")
    k, v = (torch.stack([d[i].transpose(0, 1) for d in dense]).half().cuda() for i in (0, 1))
    dense_o = scaled_dot_product_attention(q, k, v, enable_gqa=True, backend="triton")
    assert torch.allclose(o.float(), dense_o.float(), atol=2e-3, rtol=2e-3)


@pytest.mark.gpu
def test_attention_kernel_over_a_cache_past_32_bits():
    """Pages on both sides of 4 GiB from the cache's start, store and attention."""
    H, S, D = 8, 64, 128
    pages = (5 << 30) // (H * S * D * 2)
    kc, vc = (torch.empty(pages, H, S, D, dtype=torch.float16, device="cuda") for _ in range(2))
    use = [0, pages - 1, pages // 2, pages - 2, 7]
    n = 300
    gen = torch.Generator().manual_seed(3)
    key, value = (torch.randn(n, H, D, generator=gen).half() for _ in range(2))
    slots = torch.tensor([use[i // S] * S + i % S for i in range(n)])
    paged_cache_store(key.cuda(), value.cuda(), kc, vc, slots.cuda(), backend="triton")
    assert torch.equal(kc[pages - 1].cpu(), key[S:2 * S].transpose(0, 1))
    table = torch.tensor([use], dtype=torch.int32).cuda()
    q = torch.randn(1, 32, 1, D, generator=gen).half().cuda()
    o = paged_attention(q, kc, vc, table, torch.tensor([n], dtype=torch.int32).cuda(),
                        enable_gqa=True, backend="triton")
    want, bound = attention_reference(q, [[key.double(), value.double()]], D ** -0.5, torch.float16)
    limit = HALF[torch.float16] * want.abs() * 1.01 + bound * 1.01
    assert ((o.double().cpu() - want).abs() <= limit).all()


@pytest.mark.gpu
def test_attention_kernel_of_more_heads_than_a_grid_holds():
    """2^24 heads of 2^21 sequences and some, short tables: all read one page. Against calls of
    the sequences' parts."""
    B, H, S, D = (1 << 21) + 9, 8, 16, 8
    gen = torch.Generator(device="cuda").manual_seed(4)
    kc, vc = (torch.randn(2, H, S, D, dtype=torch.float16, device="cuda", generator=gen)
              for _ in range(2))
    q = torch.empty(B, H, 1, D, dtype=torch.float16, device="cuda").normal_(generator=gen)
    lens = torch.randint(0, S + 1, (B,), dtype=torch.int32, device="cuda", generator=gen)
    table = torch.ones(1, 1, dtype=torch.int32, device="cuda").expand(B, 1)
    o = paged_attention(q, kc, vc, table, lens, backend="triton")
    for a in range(0, B, 1 << 18):
        part = slice(a, min(a + (1 << 18), B))
        want = paged_attention(q[part], kc, vc, table[part], lens[part], backend="triton")
        assert torch.equal(o[part], want), a
    want, bound = attention_reference(
        q[-5:], [[t[1].transpose(0, 1)[:n].double().cpu() for t in (kc, vc)]
                 for n in lens[-5:].tolist()], D ** -0.5, torch.float16)
    assert ((o[-5:].double().cpu() - want).abs() <= HALF[torch.float16] * want.abs() * 1.01
            + bound * 1.01 + 2.0 ** -24).all()


@pytest.mark.gpu
def test_attention_kernel_refuses_what_it_cannot_serve():
    a = _attend_args("cuda")
    a["query"].requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        paged_attention(**a, backend="triton")
    assert paged_attention(**a).requires_grad  # PyTorch serves it
    with torch.no_grad():
        paged_attention(**a, backend="triton")
    with pytest.raises(RuntimeError, match="float16 and bfloat16"):
        paged_attention(**_attend_args("cuda", torch.float32), backend="triton")


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_binding_and_op_layer(native, monkeypatch):
    """The same calls through the C++ binding and without it."""
    assert _native.available(), _native.status()[1]
    if not native:
        monkeypatch.setattr(_native, "available", lambda: False)
    check_plan(lengths=ragged(37, 300, 1), new=ragged(37, 70, 2), S=16, start=2, device="cuda",
               backend="triton", pad_columns=2)
    check_store(50, 8, 128, 32, torch.float16, layout="fused", cache_layout="tokens",
                device="cuda", backend="triton")
    check_attend([700, 0, 33], 8, 2, 3, 96, 48, torch.bfloat16, layout="tokens", q_layout="tokens",
                 device="cuda", backend="triton")


# ---- a decoding loop --------------------------------------------------------------------


def decode(device, backend, dtype, steps, *, graph=False):
    """Prompts of three sequences, then ``steps`` tokens each, through plan, qk_norm_rope,
    store and attention; every output against attention in 64 bits over the keys and values so
    far. With ``graph`` the decoding step is captured once and replayed."""
    B, Hq, Hkv, D, S, M = 3, 8, 2, 64, 16, 8
    gen = torch.Generator().manual_seed(11)
    z = dict(dtype=dtype, device=device)
    i32 = dict(dtype=torch.int32, device=device)
    pages = B * M
    kc, vc = (torch.full((pages, Hkv, S, D), math.nan, **z) for _ in range(2))
    table = torch.full((B, M), -1, **i32)
    free = torch.randperm(pages, generator=gen).int().to(device)
    start, lengths = torch.zeros(1, **i32), torch.zeros(B, **i32)
    angle = torch.arange(200.0)[:, None] * 100.0 ** (-torch.arange(0, D, 2) / D)
    cos, sin = angle.cos().to(device), angle.sin().to(device)
    wq, wk = (1 + 0.2 * torch.randn(D, generator=gen)).to(**z), torch.ones(D, **z)
    history = [[] for _ in range(B)]

    def step(new, x, T, n):
        """T tokens of x [1, T, Hq + 2 Hkv, D]; attention of the newest n of each sequence."""
        p = paged_cache_plan(table, lengths, new, free, page_size=S, num_tokens=T,
                             free_start=start, backend=backend)
        q, k, v = (t.transpose(1, 2) for t in x.split([Hq, Hkv, Hkv], 2))
        q, k = qk_norm_rope(q, k, cos, sin, query_weight=wq, key_weight=wk,
                            positions=p.positions, backend=backend)
        paged_cache_store(k[0].transpose(0, 1), v[0].transpose(0, 1), kc, vc, p.slots,
                          backend=backend)
        lengths.copy_(p.lengths)
        start.copy_(p.free_start)
        last = (p.starts[1:, None].long() - n + torch.arange(n, device=device)).flatten()
        q = q[0].index_select(1, last).view(Hq, B, n, D).transpose(0, 1)
        o = paged_attention(q, kc, vc, table, lengths, enable_gqa=True, backend=backend)
        return p, q, k, v, o

    def check(result, counts):
        p, q, k, v, o = result
        at = 0
        for b, c in enumerate(counts):
            for t in range(at, at + c):
                assert p.positions[t].item() == len(history[b])
                history[b].append((k[0, :, t].cpu().clone(), v[0, :, t].cpu().clone()))
            at += c
        dense = [[torch.stack([kv[i] for kv in h]).double() for i in (0, 1)] for h in history]
        want, bound = attention_reference(q, dense, D ** -0.5, dtype)
        limit = HALF[dtype] * want.abs() * 1.01 + bound * 1.01 + 2.0 ** -24
        assert ((o.double().cpu() - want).abs() <= limit).all()

    def tokens(T):
        return torch.randn(1, T, Hq + 2 * Hkv, D, generator=gen).to(**z)

    with torch.no_grad():
        prompts = [13, 16, 40]
        check(step(torch.tensor(prompts, **i32), tokens(80), 80, 2), prompts)
        one = torch.ones(B, **i32)
        x = tokens(B)
        if graph:
            saved = [t.clone() for t in (kc, vc, table, start, lengths)]
            captured = torch.cuda.CUDAGraph()
            with torch.cuda.graph(captured):
                result = step(one, x, B, 1)
            for t, s in zip((kc, vc, table, start, lengths), saved):
                t.copy_(s)
        for _ in range(steps):
            x.copy_(tokens(B))
            if graph:
                captured.replay()
                torch.cuda.synchronize()
            else:
                result = step(one, x, B, 1)
            check(result, [1] * B)
    used = start.item()
    assert used == sum(cdiv(len(h), S) for h in history)
    assert sorted(t for t in table.flatten().tolist() if t >= 0) == sorted(free[:used].tolist())


def test_decoding_loop_torch_forms():
    decode("cpu", "torch", torch.float32, 5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_decoding_loop_kernels(dtype):
    decode("cuda", "triton", dtype, 20)


@pytest.mark.gpu
def test_decoding_loop_captured_and_replayed():
    decode("cuda", "triton", torch.bfloat16, 12, graph=True)


def run_module_example(device, dtype):
    """The step of the module's docstring as it stands, on prompts of several lengths."""
    from triton_flash_attention import paged

    code = "\n".join(line[4:] for line in paged.__doc__.splitlines() if line.startswith("    "))
    assert code.startswith("plan = paged_cache_plan(")
    B, Hq, Hkv, D, n, T, S = 3, 4, 2, 64, 2, 44, 16
    gen = torch.Generator().manual_seed(12)
    i32, z = dict(dtype=torch.int32, device=device), dict(dtype=dtype, device=device)
    new = [5, 2, 33]
    angle = torch.rand(64, D // 2, generator=gen)
    q, k, v = (torch.randn(1, h, T, D, generator=gen).to(**z) for h in (Hq, Hkv, Hkv))
    names = dict(
        torch=torch, n=n, T=T, table=torch.full((B, 4), -1, **i32), lengths=torch.zeros(B, **i32),
        new_tokens=torch.tensor(new, **i32), free_pages=torch.arange(7, -1, -1, **i32), q=q, k=k, v=v,
        cos=angle.cos().to(device), sin=angle.sin().to(device),
        key_cache=torch.zeros(8, Hkv, S, D, **z), value_cache=torch.zeros(8, Hkv, S, D, **z),
        paged_cache_plan=paged_cache_plan, paged_cache_store=paged_cache_store,
        paged_attention=paged_attention, qk_norm_rope=qk_norm_rope)
    exec(code, names)
    keys, values, dense, ends = names["k"][0], v[0], [], [5, 7, 40]
    for end, c in zip(ends, new):
        dense.append([t[:, end - c:end].transpose(0, 1).double().cpu() for t in (keys, values)])
    assert names["q"].shape == (B, Hq, n, D)
    want, bound = attention_reference(names["q"], dense, D ** -0.5, dtype)
    off = (names["out"].double().cpu() - want).abs()
    assert (off <= HALF[dtype] * want.abs() * 1.01 + bound * 1.01 + 2.0 ** -24).all()
    # the rotated queries of the newest tokens
    place = torch.tensor([c - n + j for c in new for j in range(n)])
    row = torch.tensor([e - n + j for e in ends for j in range(n)])
    x = q[0][:, row.to(device)].double().cpu()
    c, s, h = angle.cos()[place].double(), angle.sin()[place].double(), D // 2
    x = torch.cat((x[..., :h] * c - x[..., h:] * s, x[..., h:] * c + x[..., :h] * s), -1)
    got = names["q"].transpose(0, 1).flatten(1, 2).double().cpu()
    assert torch.allclose(got, x, rtol=0, atol=8 * HALF[dtype])


def test_module_example():
    run_module_example("cpu", torch.float32)


@pytest.mark.gpu
def test_module_example_on_the_kernels():
    run_module_example("cuda", torch.float16)


def test_torch_forms_compile():
    """The PyTorch forms trace as one graph."""
    a = _attend_args(dtype=torch.float32)

    def f(q, t, n):
        o = paged_attention(q, a["key_cache"], a["value_cache"], t, n, enable_gqa=True)
        return o + paged_cache_plan(t, n, n, n, page_size=16, num_tokens=4).slots.sum()

    args = (a["query"], a["page_table"], a["lengths"])
    torch._dynamo.reset()
    torch.testing.assert_close(torch.compile(f, fullgraph=True, backend="eager")(*args), f(*args))


@pytest.mark.gpu
def test_kernels_under_torch_compile():
    """Calls that the kernels serve run beside the compiled graph, with the same results."""
    a = _attend_args("cuda")
    a["key_cache"].normal_()
    a["value_cache"].normal_()
    a["query"].normal_()
    a["lengths"].fill_(20)
    cos = torch.randn(4, 16, device="cuda")

    def f(q):
        q, k = qk_norm_rope(q + 1, q - 1, cos, cos)
        return paged_attention(q * 2, a["key_cache"], a["value_cache"], a["page_table"],
                               a["lengths"], enable_gqa=True) + k

    with torch.no_grad():
        torch._dynamo.reset()
        assert torch.equal(torch.compile(f, backend="eager")(a["query"]), f(a["query"]))


@pytest.mark.gpu
def test_kernels_from_two_threads_on_two_streams():
    """Calls at once, each with tensors and a workspace of its own."""
    import threading

    failures = []

    def work(seed):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for i in range(4):
                    check_attend([2500, 40, 1200], 8, 2, 1, 64, 16, torch.float16,
                                 seed=10 * seed + i, device="cuda", backend="triton")
                    check_plan(ragged(70, 300, seed), ragged(70, 9, i), 16, device="cuda",
                               backend="triton")
                stream.synchronize()
        except BaseException as e:  # noqa: BLE001 - raised below
            failures.append(e)

    threads = [threading.Thread(target=work, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures[0]


@pytest.mark.gpu
def test_two_captured_steps_replayed_in_turn():
    """Two graphs of attention calls that share torch's pool: each keeps its own partials."""
    cases = [make_paged([3000, 17], 2, 16, 64, torch.float16, device="cuda", seed=s) for s in (1, 2)]
    gen = torch.Generator().manual_seed(4)
    q = torch.randn(2, 8, 1, 64, generator=gen).half().cuda()
    pool = torch.cuda.graph_pool_handle()
    graphs, outs, wants = [], [], []
    for views, table, lens, dense in cases:
        paged_attention(q, *views, table, lens, enable_gqa=True, backend="triton")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(paged_attention(q, *views, table, lens, enable_gqa=True, backend="triton"))
        graphs.append(g)
    for i in range(3):
        q.copy_(torch.randn(2, 8, 1, 64, generator=gen).half())
        wants = [paged_attention(q, *v, t, n, enable_gqa=True, backend="triton")
                 for v, t, n, _ in cases]
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, wants)), i


@pytest.mark.gpu
def test_kernels_on_another_stream():
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        decode("cuda", "triton", torch.float16, 2)
    side.synchronize()
