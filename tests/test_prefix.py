"""Attention over the paged cache whose groups of sequences share prefixes, against the plain
implementation in 64 bits and with the element-wise tolerance of test_paged.py: the PyTorch form on
the CPU and the gfx950 kernels on the GPU. The kernels' pieces are joined by weights in float32,
which adds a few 2^-24 of A, far inside the 4 d A of that bound (d is at least 136 2^-24)."""

from __future__ import annotations

import math
import random

import pytest
import torch
from test_paged import F32, HALF, attention_reference, cdiv, ragged

from triton_flash_attention import paged_attention, paged_prefix_attention


def make_shared(sizes, prefix, lengths, Hkv, S, D, dtype, *, seed=0, layout="heads", M=None,
                fill=math.nan, device="cpu", spread=1.0):
    """A cache whose groups' prefixes lie in the pages of their first sequences alone: the other
    rows name no page for whole pages of the prefix, and the cache holds ``fill`` wherever no token
    lies. Returns the caches, the table, the groups' starts, and the dense keys and values
    [n, Hkv, D] of each sequence (float64)."""
    gen = torch.Generator().manual_seed(seed)
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + n)
    leader, front = list(range(len(lengths))), [0] * len(lengths)
    for g, n in enumerate(sizes):
        for b in range(starts[g], starts[g + 1]):
            if n > 1:
                leader[b], front[b] = starts[g], max(0, min(prefix[g], lengths[starts[g]]))
    M = M or max(1, *(cdiv(n, S) for n in lengths))
    pages = sum(cdiv(n, S) for n in lengths) + 3
    order = torch.randperm(pages, generator=gen).tolist()
    shape = (pages, S, Hkv, D) if layout == "tokens" else (pages, Hkv, S, D)
    caches = [torch.full(shape, fill).to(dtype) for _ in range(2)]
    views = [c.transpose(1, 2) if layout == "tokens" else c for c in caches]
    table, dense = torch.full((len(lengths), M), -9, dtype=torch.int32), []
    for b, n in enumerate(lengths):
        kv = [(torch.randn(n, Hkv, D, generator=gen) * spread).to(dtype) for _ in range(2)]
        first = front[b] if leader[b] != b else 0  # the sequence's first key in pages of its own
        for j in range(first // S, cdiv(n, S)):
            if n <= first:
                break
            table[b, j] = page = order.pop()
            lo, hi = max(j * S, first), min((j + 1) * S, n)
            for c, t in zip(views, kv):
                c[page, :, lo - j * S:hi - j * S] = t[lo:hi].transpose(0, 1)
        if first:
            kv = [torch.cat((d[:min(first, n)].to(dtype), t[first:]))
                  for d, t in zip(dense[leader[b]], kv)]
        dense.append([t.double() for t in kv])
    caches = [c.to(device) for c in caches]
    views = [c.transpose(1, 2) if layout == "tokens" else c for c in caches]
    return views, table.to(device), torch.tensor(starts, dtype=torch.int32, device=device), dense


def within(o, want, bound, dtype):
    off = (o.double().cpu() - want).abs()
    limit = HALF[dtype] * want.abs() * 1.01 + bound * 1.01 + 2.0 ** -24
    assert bool((off <= limit).all()), f"{(off / limit).max().item():.3f} of the bound"


def check_prefix(sizes, prefix, lengths, Hq, Hkv, N, D, S, dtype, *, scale=None, seed=0,
                 device="cpu", backend="torch", q_layout="heads", q_spread=1.0, **cache):
    views, table, starts, dense = make_shared(sizes, prefix, lengths, Hkv, S, D, dtype, seed=seed,
                                              device=device, **cache)
    gen = torch.Generator().manual_seed(seed + 1)
    B = len(lengths)
    if q_layout == "tokens":
        q = (torch.randn(B, N, Hq + 3, D, generator=gen) * q_spread).to(dtype).to(device)
        q = q[:, :, 1:Hq + 1].transpose(1, 2)
    else:
        q = (torch.randn(B, Hq, N, D, generator=gen) * q_spread).to(dtype).to(device)
    ints = [torch.tensor(v, dtype=torch.int32, device=device) for v in (lengths, prefix)]
    o = paged_prefix_attention(q, *views, table, ints[0], starts, ints[1], scale=scale,
                               enable_gqa=Hq != Hkv, backend=backend)
    want, bound = attention_reference(q, dense, D ** -0.5 if scale is None else scale, dtype)
    assert o.shape == want.shape and o.is_contiguous() and o.dtype == dtype
    within(o, want, bound, dtype)
    return o


CASES = [
    # sizes, prefixes, lengths, Hq, Hkv, N, D, S
    ([1], [0], [1], 1, 1, 1, 32, 16),
    ([2], [1], [1, 2], 1, 1, 1, 32, 16),
    ([3], [32], [33, 40, 70], 4, 2, 1, 64, 16),
    ([2, 3], [16, 40], [17, 31, 64, 41, 100], 8, 2, 1, 128, 16),
    # prefixes that end inside a page, a half unit, a unit
    ([4], [37], [38, 50, 37, 90], 6, 2, 1, 64, 32),
    ([2, 2, 2], [5, 15, 17], [9, 21, 16, 40, 18, 33], 4, 4, 1, 40, 48),
    # sequences as short as the prefix, shorter, empty; prefixes longer than the first sequence
    ([5], [60], [70, 60, 31, 0, 1], 4, 2, 2, 32, 16),
    ([3], [500], [40, 90, 20], 4, 1, 3, 80, 16),
    ([2, 2], [30, 30], [0, 50, 20, 0], 2, 2, 1, 64, 16),
    ([2], [-4], [20, 30], 2, 1, 1, 64, 16),
    # groups of none, of one; sequences outside all groups
    ([0, 3, 0, 1], [9, 16, 3, 20], [30, 20, 17, 40], 4, 2, 1, 32, 16),
    ([2], [32], [40, 50, 60, 7], 4, 2, 1, 64, 16),
    ([], [], [33, 2], 2, 1, 1, 32, 16),
    # several tokens: rows of one sequence in several tiles
    ([3], [64], [90, 70, 133], 16, 1, 9, 32, 16),
    ([2], [100], [150, 104], 32, 2, 5, 128, 64),
]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_torch_form(case, dtype):
    check_prefix(*case, dtype)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.7])
def test_torch_form_scales(scale):
    check_prefix([2, 2], [20, 16], [40, 21, 17, 30], 4, 2, 2, 32, 16, torch.float32, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
@pytest.mark.parametrize("case", CASES)
def test_kernel(case, layout, dtype):
    check_prefix(*case, dtype, layout=layout, q_layout=layout, device="cuda", backend="triton")


def many(sizes, lo, hi, seed):
    """Prefixes and lengths for groups of these sizes."""
    rng = random.Random(seed)
    prefix = [rng.randint(lo, hi) for _ in sizes]
    lengths = [max(1, p + rng.choice([0, 1, rng.randint(-5, 40), rng.randint(1, hi)]))
               for p, n in zip(prefix, sizes) for _ in range(n)]
    return sizes, prefix, lengths


WORK_GROUPS = [
    # one group over the whole chip
    (*many([7], 3001, 3001, 1), 32, 8, 1, 128, 16),
    (*many([40], 700, 700, 2), 16, 4, 1, 64, 32),        # two tiles of rows
    (*many([33], 260, 260, 3), 8, 2, 5, 96, 16),          # 660 rows
    (*many([2] * 30, 40, 900, 4), 8, 8, 1, 64, 16),
    (*many([1, 3, 2, 9, 1, 1, 5], 1, 1500, 5), 4, 2, 2, 32, 48),
    (*many([2], 20000, 20000, 6), 2, 1, 17, 32, 16),      # many units a work-group
    (*many([300], 64, 64, 7), 2, 2, 1, 32, 16),           # more sequences than threads
    (*many([2] * 400, 1, 60, 8), 2, 1, 1, 64, 16),        # and groups
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", WORK_GROUPS)
def test_kernel_over_work_groups(case, dtype):
    M = cdiv(max(case[2]), case[7]) + 3
    o = check_prefix(*case, dtype, device="cuda", backend="triton", M=M)
    assert torch.equal(o, check_prefix(*case, dtype, device="cuda", backend="triton", M=M))


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(16))
def test_kernel_random(seed):
    rng = random.Random(100 + seed)
    Hkv = rng.choice([1, 2, 3, 5])
    S, G = rng.choice([16, 32, 48, 80]), rng.choice([1, 1, 2, 7, 33])
    sizes = [rng.randint(0, rng.choice([1, 4, 40]) if G < 8 else 5) for _ in range(G)]
    hi = rng.choice([60, 700, 3000 if G < 8 else 500])
    sizes, prefix, lengths = many(sizes, rng.choice([0, hi // 2]), hi, seed)
    lengths += ragged(rng.choice([0, 3]) or 1 - min(1, len(lengths)), hi, seed)  # outside the groups
    check_prefix(sizes, prefix, lengths, Hkv * rng.choice([1, 2, 4, 6]), Hkv, rng.choice([1, 1, 2, 3]),
                 rng.choice([8, 32, 48, 64, 104, 128]), S, rng.choice([torch.float16, torch.bfloat16]),
                 layout=rng.choice(["heads", "tokens"]), q_layout=rng.choice(["heads", "tokens"]),
                 M=max(cdiv(max(lengths), S), rng.choice([1, cdiv(9000, S)])), seed=seed,
                 device="cuda", backend="triton")


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.3, 1.7, 1e-40])
def test_kernel_scales(scale):
    check_prefix([2, 2], [300, 16], [400, 301, 17, 30], 4, 2, 2, 64, 16, torch.float16, scale=scale,
                 device="cuda", backend="triton")


@pytest.mark.gpu
def test_kernel_large_scores():
    """Scores in the thousands: one key takes all the weight, in the prefix or behind it."""
    check_prefix([6], [777], [1000, 777, 778, 900, 2000, 1500], 8, 2, 1, 64, 16, torch.bfloat16,
                 q_spread=30.0, device="cuda", backend="triton")


@pytest.mark.gpu
@pytest.mark.parametrize("fill", [math.inf, -math.inf, 65504.0])
def test_kernel_never_sees_what_lies_elsewhere(fill):
    check_prefix([4, 1], [37, 0], [70, 38, 50, 37, 20], 8, 2, 1, 128, 32, torch.float16, fill=fill,
                 device="cuda", backend="triton")


def bad_rows(device, backend, dtype):
    """Lengths and pages that do not exist make the sequences NaN that need them, and no other."""
    sizes, prefix, lengths = [3, 2, 3], [32, 32, 32], [40, 50, 36, 40, 64, 50, 20, 60]
    views, table, starts, dense = make_shared(sizes, prefix, lengths, 2, 16, 64, dtype, M=4, fill=0.0,
                                              device=device)
    q = torch.randn(8, 4, 1, 64, generator=torch.Generator().manual_seed(3)).to(dtype).to(device)
    pages = views[0].shape[0]
    lens, pre = (torch.tensor(v, dtype=torch.int32, device=device) for v in (lengths, prefix))
    table[1, 3] = pages          # of sequence 1's own keys
    lens[4] = 65                 # more than its row holds
    table[5, 1] = -2             # of a prefix: keys 16 to 31
    lens[6] = 16                 # which a short sequence does not need
    table[0, 3] = 1 << 30        # behind the length: not looked at
    o = paged_prefix_attention(q, *views, table, lens, starts, pre, enable_gqa=True,
                               backend=backend).cpu()
    dense[6] = [t[:16] for t in dense[6]]
    want, _ = attention_reference(q, dense, 0.125, dtype)
    for b in range(8):
        if b in (1, 4, 5, 7):
            assert o[b].isnan().all(), b
        else:
            assert torch.allclose(o[b].double(), want[b], atol=2e-2), b
    # an invalid first sequence has no prefix to share, and spoils no other
    lens[0] = -1
    table[1:3, :2] = table[0, :2].clone()
    o = paged_prefix_attention(q, *views, table, lens, starts, pre, enable_gqa=True,
                               backend=backend).cpu()
    assert o[0].isnan().all() and o[1].isnan().all()
    assert torch.allclose(o[2].double(), want[2], atol=2e-2)
    # starts that do not ascend within the batch
    for bad in ([0, 3, 2, 8], [-1, 3, 5, 8], [0, 3, 5, 9]):
        s = torch.tensor(bad, dtype=torch.int32, device=device)
        assert paged_prefix_attention(q, *views, table, lens, s, pre, enable_gqa=True,
                                      backend=backend).isnan().all()


def test_torch_form_bad_rows():
    bad_rows("cpu", "torch", torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_kernel_bad_rows(dtype):
    bad_rows("cuda", "triton", dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [896, 32768])
def test_kernel_counts_the_many_small_weights_of_long_prefixes(n, dtype):
    """The prefix's first key and each sequence's last have the largest score, 18 above all others:
    2^-26 of their weight each, and the only ones with a value."""
    S, D, B = 16, 32, 40
    k, v = (torch.zeros(2, 1, S, D, dtype=dtype, device="cuda") for _ in range(2))
    k[1, 0, 0, 0], v[:] = 18.0, 1.0
    v[1, 0, 0] = 0.0
    table = torch.zeros(B, n // S + 1, dtype=torch.int32, device="cuda")
    table[:, 0] = table[:, -1] = 1
    q = torch.zeros(B, 1, 1, D, dtype=dtype, device="cuda")
    q[..., 0] = 1.0
    i32 = dict(dtype=torch.int32, device="cuda")
    o = paged_prefix_attention(q, k, v, table, torch.full((B,), n + 1, **i32),
                               torch.tensor([0, B], **i32), torch.tensor([n], **i32), scale=1.0,
                               backend="triton").double().cpu()
    small = (n - 1) * math.exp(-18.0)
    want = small / (2 + small)
    d = (136 + 8) * 18 * F32
    bound = want * (2 * HALF[dtype] + n * F32 + 4 * d) + (
        n / 2 * 2.0 ** -32 + 2.0 ** -25 if dtype == torch.float16 else 0)
    assert float((o - want).abs().max()) <= bound


LARGE = [("random", 300), ("equal", 300), ("equal", 9000), ("grow", 1200)]


@pytest.mark.gpu
@pytest.mark.parametrize(("kind", "n"), LARGE)
def test_kernel_large_values(kind, n):
    """Values of up to 2^127, whose sums have no room in float32."""
    sizes, prefix, lengths = [3], [n], [n + 40, n + 1, n]
    S, D, Hq, Hkv, N, dtype = 16, 32, 4, 2, 2, torch.bfloat16
    views, table, starts, dense = make_shared(sizes, prefix, lengths, Hkv, S, D, dtype, seed=6)
    views[1].abs_().mul_(2.0 ** 124)
    for b, (k, v) in enumerate(dense):
        v.abs_().mul_(2.0 ** 124)
        at = torch.arange(lengths[b])
        if kind == "equal":
            k.zero_()
        elif kind == "grow":
            k.zero_()[:, :, 0] = (at // 40 * 4.0).clamp(max=120.0)[:, None]
        row = torch.where(at < n, table[0].long()[at // S], table[b].long()[at // S])
        views[0][row, :, at % S] = k.to(dtype)
    q = torch.randn(3, Hq, N, D, generator=torch.Generator().manual_seed(7)).to(dtype)
    if kind == "grow":
        q[..., 0] = 1.0
    ints = [torch.tensor(t, dtype=torch.int32, device="cuda") for t in (lengths, prefix)]
    o = paged_prefix_attention(q.cuda(), *(t.cuda() for t in views), table.cuda(), ints[0],
                               starts.cuda(), ints[1], scale=1.0, enable_gqa=True, backend="triton")
    want, bound = attention_reference(q, dense, 1.0, dtype)
    limit = HALF[dtype] * want.abs() * 1.01 + bound * 1.01
    assert bool(((o.double().cpu() - want).abs() <= limit).all())


def test_groups_of_one_are_the_plain_attention():
    views, table, starts, _ = make_shared([1, 1], [9, 9], [40, 21], 2, 16, 32, torch.float32, fill=0.0)
    q = torch.randn(2, 4, 1, 32)
    lens, pre = (torch.tensor(v, dtype=torch.int32) for v in ([40, 21], [9, 9]))
    assert torch.allclose(
        paged_prefix_attention(q, *views, table, lens, starts, pre, enable_gqa=True),
        paged_attention(q, *views, table, lens, enable_gqa=True), atol=1e-6)


def _args(device="cpu", dtype=torch.float16):
    z = dict(dtype=dtype, device=device)
    i = dict(dtype=torch.int32, device=device)
    return dict(query=torch.zeros(2, 4, 1, 32, **z), key_cache=torch.zeros(4, 2, 16, 32, **z),
                value_cache=torch.zeros(4, 2, 16, 32, **z), page_table=torch.zeros(2, 3, **i),
                lengths=torch.ones(2, **i), group_starts=torch.tensor([0, 2], **i),
                prefix_lengths=torch.ones(1, **i), enable_gqa=True)


@pytest.mark.parametrize(("change", "error", "message"), [
    (dict(backend="x"), ValueError, "backend"),
    (dict(enable_gqa=False), ValueError, "enable_gqa=True"),
    (dict(scale=float("nan")), ValueError, "scale"),
    (dict(query=torch.zeros(2, 4, 1, 64).half()), ValueError, "head dimensions"),
    (dict(page_table=torch.zeros(3, 3).int()), ValueError, "a row for each sequence"),
    (dict(lengths=torch.ones(2).long()), ValueError, "lengths must be int32"),
    (dict(group_starts=[0, 2]), TypeError, "group_starts"),
    (dict(group_starts=torch.zeros(3).int()), ValueError, "group_starts must have shape"),
    (dict(group_starts=torch.zeros(2)), ValueError, "group_starts must be int32"),
    (dict(prefix_lengths=torch.zeros(1, 1).int()), ValueError, "prefix_lengths must have shape"),
    (dict(prefix_lengths=torch.zeros(1).long()), ValueError, "prefix_lengths must be int32"),
    (dict(backend="triton"), RuntimeError, "CUDA tensor"),
])
def test_refusals(change, error, message):
    with pytest.raises(error, match=message):
        paged_prefix_attention(**{**_args(), **change})
