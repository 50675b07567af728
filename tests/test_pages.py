"""Pages that sequences share: forks, copies and compaction of the paged cache against walks over
lists (whole numbers and copied values exactly), the PyTorch forms on the CPU and the gfx950
kernels on the GPU, and beam decoding that runs them with the plan, the store and the attention
over shared prefixes."""

from __future__ import annotations

import math
import random

import pytest
import torch
from test_paged import attention_reference, cdiv, ragged
from test_prefix import within

from triton_flash_attention import (paged_cache_compact, paged_cache_copy, paged_cache_fork,
                                    paged_cache_plan, paged_cache_store, paged_prefix_attention)


def ints(v, device="cpu"):
    return torch.tensor(v, dtype=torch.int32, device=device)


# ---- fork -------------------------------------------------------------------------------


def fork_reference(table, lengths, parents, free, shares, start, S):
    """The fork by a walk over the rows: (table, free, shares, lengths, sources, targets, tokens,
    start), all lists."""
    table, free, shares = [r[:] for r in table], free[:], shares[:]
    B, P, start = len(table), len(shares), min(max(start, 0), len(free))
    M = len(table[0]) if B else 1
    lengths = [max(n, 0) for n in lengths]
    before = [row[:min(cdiv(n, S), M)] for row, n in zip(table, lengths)]
    sources, targets, tokens, after = [-1] * B, [-1] * B, [0] * B, []
    goes_on = {p: p for p in parents if 0 <= p < B and parents[p] == p}
    new, taken = [], 0
    for b, p in enumerate(parents):
        if not 0 <= p < B:
            after.append([])
            new.append(0)
            continue
        row, n = before[p][:], lengths[p]
        begun = n % S if cdiv(n, S) <= M else 0
        if begun and goes_on.setdefault(p, b) != b and 0 <= row[-1] < P:
            place = start + taken
            sources[b], tokens[b] = row[-1], begun
            targets[b] = row[-1] = free[place] if place < len(free) else -1
            taken += 1
        after.append(row)
        new.append(n)
    holders = [s + 1 for s in shares]
    touched = set()
    for rows, step in ((before, -1), (after, 1)):
        for b, row in enumerate(rows):
            for j, page in enumerate(row):
                copied = step > 0 and targets[b] == page and j == len(row) - 1 and sources[b] >= 0
                if 0 <= page < P and not copied:
                    holders[page] += step
                    touched.add(page)
    gone = sorted(p for p in touched if holders[p] == 0)
    for p in touched:
        shares[p] = max(holders[p] - 1, 0)
    first = start + min(taken, len(free) - start) - len(gone)
    for k, p in enumerate(gone):
        if first + k >= 0:
            free[first + k] = p
    for b, row in enumerate(after):
        table[b][:len(row)] = row
    return table, free, shares, new, sources, targets, tokens, max(first, 0)


def shared_rows(lengths, S, seed, *, M=None, groups=3, spare=None):
    """Rows of which neighbours share whole pages, the counts, and the free pages."""
    rng = random.Random(seed)
    held = [cdiv(max(n, 0), S) for n in lengths]
    M = M or max([1, *held])
    pages = list(range(sum(held) + (len(lengths) + 4 if spare is None else spare)))
    rng.shuffle(pages)
    shares, table = [0] * len(pages), []
    for b, h in enumerate(held):
        h = min(h, M)
        row = [-7] * M
        both = min(h, held[b - 1], max(lengths[b], 0) // S, max(lengths[b - 1], 0) // S) if b % groups else 0
        same = rng.randint(0, both)
        for j in range(h):
            if j < same:
                row[j] = table[b - 1][j]
                shares[row[j]] += 1
            else:
                row[j] = pages.pop()
        table.append(row)
    return table, shares, pages


def check_fork(lengths, parents, S, *, M=None, seed=0, device="cpu", backend="torch", start=None,
               free=None, pad_columns=0, change=None, **rows):
    table, shares, pages = shared_rows(lengths, S, seed, M=M, **rows)
    if change:
        change(table)
    # every page has a place in the list
    pages = [-3] * (len(shares) - len(pages)) + pages if free is None else free(pages)
    first = len(shares) - sum(p >= 0 for p in pages) if start is None and free is None else start
    want = fork_reference(table, lengths, parents, pages, shares, first or 0, S)
    width = len(table[0]) if table else 1
    t = torch.full((len(lengths), width + pad_columns), -9, dtype=torch.int32, device=device)
    t = t[:, :width]
    if lengths:
        t.copy_(ints(table, device))
    f, s = ints(pages, device), ints(shares, device)
    versions = [x._version for x in (t, f, s)]
    got = paged_cache_fork(t, ints(lengths, device), ints(parents, device), f, s, page_size=S,
                           free_start=None if first is None else ints([first], device),
                           backend=backend)
    assert not lengths or all(x._version > v for x, v in zip((t, f, s), versions))
    for name, a, b in zip(("lengths", "sources", "targets", "tokens"), got, want[3:7]):
        assert a.dtype == torch.int32 and a.tolist() == b, name
    assert t.tolist() == want[0] and f.tolist() == want[1] and s.tolist() == want[2]
    assert got.free_start.tolist() == [want[7]]


def some_parents(B, seed, ends=0.2):
    rng = random.Random(seed)
    return [-1 if rng.random() < ends else rng.randrange(B) for _ in range(B)]


def bad_entries(table):
    table[0][0] = -5
    table[1][-1] = 1 << 20
    table[2][0] = 1 << 30


FORKS = [
    dict(lengths=[5], parents=[0], S=16),                       # nothing changes
    dict(lengths=[5], parents=[-1], S=16),                      # a sequence ends
    dict(lengths=[20, 0, 0, 0], parents=[0, 0, 0, 0], S=16),    # a prompt is sampled four times
    dict(lengths=[32, 0, 0], parents=[0, 0, 0], S=16),          # ... which fills its pages
    dict(lengths=[20, 30, 40, 50], parents=[3, 2, 1, 0], S=16),  # rows change places
    dict(lengths=[40, 41, 33, 50], parents=[1, 1, 1, 2], S=16),  # beams
    dict(lengths=[40, 41, 33, 50], parents=[2, 1, 1, 1], S=32),
    dict(lengths=[], parents=[], S=16),
    dict(lengths=[0, 0], parents=[1, 0], S=16),
    dict(lengths=[3, -4, 70], parents=[1, 2, 5], S=16),         # no such parent; a negative length
    dict(lengths=ragged(37, 300, 1), parents=some_parents(37, 2), S=16),
    dict(lengths=ragged(37, 300, 1), parents=some_parents(37, 3, 0.9), S=48),
    dict(lengths=[100, 50, 3], parents=[0, 0, 0], S=16, M=2),   # longer than the row
    # the free pages run out; there is no list; a start outside it
    dict(lengths=[20, 0, 0, 0], parents=[0, 0, 0, 0], S=16, free=lambda p: p[:2], start=0),
    dict(lengths=[20, 0, 40], parents=[0, 0, -1], S=16, free=lambda p: [], start=0),
    dict(lengths=[20, 0, 40], parents=[0, 0, -1], S=16, start=1000),
    dict(lengths=[20, 0, 40], parents=[0, 0, -1], S=16, start=-2),
    dict(lengths=[20, 0, 40], parents=[0, 0, -1], S=16, free=lambda p: p),
    dict(lengths=[20, 30, 40, 50], parents=[1, 1, 0, 0], S=16, change=bad_entries, groups=1),
    dict(lengths=[20, 30, 40, 50], parents=[3, 3, -1, 2], S=16, change=bad_entries, groups=1),
]


@pytest.mark.parametrize("case", FORKS)
def test_fork_torch_form(case):
    check_fork(**case)


@pytest.mark.gpu
@pytest.mark.parametrize("case", FORKS)
def test_fork_kernel(case):
    check_fork(**case, device="cuda", backend="triton")


@pytest.mark.gpu
@pytest.mark.parametrize("case", [
    dict(lengths=ragged(700, 90, 3), parents=some_parents(700, 4), S=16, pad_columns=3),
    dict(lengths=ragged(2500, 40, 5), parents=some_parents(2500, 6), S=16),   # rounds of 1024
    dict(lengths=ragged(9, 40000, 7), parents=some_parents(9, 8), S=16),      # columns in parts
    dict(lengths=[300000, 17, 200000], parents=[1, 0, 0], S=16),
    dict(lengths=ragged(300, 2000, 9), parents=some_parents(300, 10, 0.7), S=32, spare=40000),
    dict(lengths=[33] * 600, parents=[7] * 600, S=32),
])
def test_fork_kernel_over_blocks(case):
    check_fork(**case, device="cuda", backend="triton")


def chain(device, backend, seed):
    """Steps of forks and plans from an empty cache: after each, what the walk says, and every page
    is free or held as often as its count says."""
    rng = random.Random(seed)
    S, B, M, P = 16, 9, 12, 9 * 12 + 9
    table, lengths = ints([[-1] * M] * B, device), ints([0] * B, device)
    free, shares, start = ints(list(range(P)), device), ints([0] * P, device), ints([0], device)
    for step in range(25):
        lens = lengths.tolist()
        parents = [rng.choice([b, b, rng.randrange(B), -1 if rng.random() < 0.3 else b]) for b in range(B)]
        want = fork_reference(table.tolist(), lens, parents, free.tolist(), shares.tolist(),
                              int(start), S)
        fork = paged_cache_fork(table, lengths, ints(parents, device), free, shares, page_size=S,
                                free_start=start, backend=backend)
        assert [t.tolist() for t in (table, free, shares)] == list(want[:3])
        assert [t.tolist() for t in fork] == [*want[3:7], [want[7]]]
        new = ints([min(rng.randint(0, 20), M * S - n) for n in want[3]], device)
        plan = paged_cache_plan(table, fork.lengths, new, free, page_size=S, num_tokens=256,
                                free_start=fork.free_start, backend=backend)
        lengths, start = plan.lengths, plan.free_start
        held = [0] * P
        for row, n in zip(table.tolist(), lengths.tolist()):
            for page in row[:cdiv(n, S)]:
                held[page] += 1
        left = free.tolist()[int(start):]
        assert len(set(left)) == len(left)
        counts = shares.tolist()
        for p in range(P):
            assert (held[p] == 0) == (p in left), (step, p)
            assert counts[p] == max(held[p] - 1, 0), (step, p)


@pytest.mark.parametrize("seed", range(3))
def test_fork_and_plan_torch_form(seed):
    chain("cpu", "torch", seed)


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(6))
def test_fork_and_plan_kernels(seed):
    chain("cuda", "triton", seed)


@pytest.mark.gpu
def test_fork_kernel_is_the_same_every_time():
    B, S = 500, 16
    lengths, parents = ragged(B, 900, 1), some_parents(B, 2, 0.6)
    table, shares, pages = shared_rows(lengths, S, 3)
    pages = [-1] * (len(shares) - len(pages)) + pages
    first = None
    for _ in range(6):
        t, f, s = (ints(v, "cuda") for v in (table, pages, shares))
        out = paged_cache_fork(t, ints(lengths, "cuda"), ints(parents, "cuda"), f, s, page_size=S,
                               free_start=ints([sum(p < 0 for p in pages)], "cuda"), backend="triton")
        got = [x.tolist() for x in (t, f, s, *out)]
        first = first or got
        assert got == first


def _fork_args():
    i = torch.int32
    return dict(page_table=torch.zeros(2, 4, dtype=i), lengths=torch.zeros(2, dtype=i),
                parents=torch.zeros(2, dtype=i), free_pages=torch.arange(8, dtype=i),
                page_shares=torch.zeros(9, dtype=i), page_size=16)


@pytest.mark.parametrize(("change", "error", "message"), [
    (dict(backend="x"), ValueError, "backend"),
    (dict(page_table=torch.zeros(2, 4)), ValueError, "page_table must be int32"),
    (dict(page_table=torch.zeros(1, 4, dtype=torch.int32).expand(2, 4)), ValueError, "overlap"),
    (dict(page_size=24), ValueError, "multiple of 16"),
    (dict(lengths=torch.zeros(2, dtype=torch.int64)), ValueError, "lengths must be int32"),
    (dict(parents=torch.zeros(3, dtype=torch.int32)), ValueError, "parents must have shape"),
    (dict(parents=[0, 1]), TypeError, "parents"),
    (dict(free_pages=torch.zeros(2, 2, dtype=torch.int32)), ValueError, "free_pages"),
    (dict(free_pages=torch.zeros(1, dtype=torch.int32).expand(4)), ValueError, "expanded"),
    (dict(page_shares=torch.zeros(4)), ValueError, "page_shares must be int32"),
    (dict(page_shares=torch.zeros(0, dtype=torch.int32)), ValueError, "at least one page"),
    (dict(free_start=torch.zeros(2, dtype=torch.int32)), ValueError, "free_start"),
    (dict(free_start=3), TypeError, "free_start"),
    (dict(backend="triton"), RuntimeError, "CUDA tensor"),
])
def test_fork_refusals(change, error, message):
    with pytest.raises(error, match=message):
        paged_cache_fork(**{**_fork_args(), **change})


@pytest.mark.gpu
def test_fork_kernel_refuses_lists_it_cannot_write():
    a = {n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in _fork_args().items()}
    odd = torch.arange(16, dtype=torch.int32, device="cuda")[::2]
    with pytest.raises(RuntimeError, match="must be contiguous"):
        paged_cache_fork(**{**a, "free_pages": odd}, backend="triton")
    with pytest.raises(RuntimeError, match="rows of page_table"):
        paged_cache_fork(**{**a, "page_table": torch.zeros(2, 8, dtype=torch.int32, device="cuda")
                            [:, ::2]}, backend="triton")


# ---- copy -------------------------------------------------------------------------------


def check_copy(n, pages, H, D, S, dtype, *, layout="heads", part=True, device="cpu",
               backend="torch", seed=0):
    gen = torch.Generator().manual_seed(seed)
    shape = (pages, S, H, D) if layout == "tokens" else (pages, H, S, D)
    caches = [torch.randn(shape, generator=gen).to(dtype).to(device) for _ in range(2)]
    views = [c.transpose(1, 2) if layout == "tokens" else c for c in caches]
    order = torch.randperm(pages, generator=gen).int()
    sources, targets = order[:n].clone(), order[n:2 * n].clone()
    for i, (a, b) in enumerate([(-1, -1), (-1, 0), (0, -1), (pages, 0), (0, pages), (1 << 30, -9)]):
        if 4 * i + 3 < n:  # left out
            sources[4 * i + 3] = sources[4 * i + 3] if a == 0 else a
            targets[4 * i + 3] = targets[4 * i + 3] if b == 0 else b
    tokens = torch.randint(-2, S + 3, (n,), generator=gen).int() if part else None
    want = [v.clone() for v in views]
    for i, (a, b) in enumerate(zip(sources.tolist(), targets.tolist())):
        if 0 <= a < pages and 0 <= b < pages:
            k = S if tokens is None else min(max(int(tokens[i]), 0), S)
            for w in want:
                w[b, :, :k] = w[a, :, :k]
    version = views[0]._version
    paged_cache_copy(*views, sources.to(device), targets.to(device),
                     tokens=None if tokens is None else tokens.to(device), backend=backend)
    assert all(torch.equal(a, b) for a, b in zip(views, want))
    assert n == 0 or views[0]._version > version


COPIES = [
    # pairs, pages, heads, head size, page size
    (1, 2, 1, 8, 16),
    (0, 3, 2, 64, 16),
    (7, 30, 2, 64, 16),
    (30, 61, 3, 40, 48),
    (25, 60, 8, 128, 32),
    (26, 52, 5, 80, 16),
]


@pytest.mark.parametrize("part", [False, True])
@pytest.mark.parametrize("case", COPIES)
def test_copy_torch_form(case, part):
    check_copy(*case, torch.bfloat16, part=part, layout="tokens" if case[0] % 2 else "heads")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("part", [False, True])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
@pytest.mark.parametrize("case", COPIES + [(300, 700, 16, 96, 64), (900, 1800, 1, 32, 16)])
def test_copy_kernel(case, layout, part, dtype):
    check_copy(*case, dtype, layout=layout, part=part, device="cuda", backend="triton", seed=case[0])


@pytest.mark.gpu
def test_copy_kernel_of_caches_with_gaps():
    """Rows and heads that do not lie side by side: views of wider tensors."""
    wide = [torch.randn(9, 3, 20, 72, device="cuda").half() for _ in range(2)]
    views = [w[:, 1:, 2:18, 8:48] for w in wide]
    want = [w.clone() for w in wide]
    for w in want:
        w[4, 1:, 2:18, 8:48] = w[7, 1:, 2:18, 8:48]
        w[0, 1:, 2:5, 8:48] = w[3, 1:, 2:5, 8:48]
    paged_cache_copy(*views, ints([7, 3], "cuda"), ints([4, 0], "cuda"), tokens=ints([16, 3], "cuda"),
                     backend="triton")
    assert all(torch.equal(a, b) for a, b in zip(wide, want))


@pytest.mark.gpu
def test_copy_kernel_past_32_bits():
    """Pages whose addresses differ by more than 2^32 bytes."""
    caches = [torch.empty(40000, 1, 1024, 64, dtype=torch.float16, device="cuda") for _ in range(2)]
    for c in caches:
        c[39999].normal_()
        c[3].zero_()
    paged_cache_copy(*caches, ints([39999], "cuda"), ints([3], "cuda"), backend="triton")
    assert all(torch.equal(c[3], c[39999]) for c in caches)


_SAME = torch.zeros(4, 2, 16, 32).half()


def _copy_args(device="cpu", dtype=torch.float16):
    z = dict(dtype=dtype, device=device)
    return dict(key_cache=torch.zeros(4, 2, 16, 32, **z), value_cache=torch.zeros(4, 2, 16, 32, **z),
                sources=ints([0], device), targets=ints([1], device))


@pytest.mark.parametrize(("change", "error", "message"), [
    (dict(backend="x"), ValueError, "backend"),
    (dict(value_cache=torch.zeros(5, 2, 16, 32).half()), ValueError, "same shape"),
    (dict(key_cache=torch.zeros(4, 2, 24, 32).half(), value_cache=torch.zeros(4, 2, 24, 32).half()),
     ValueError, "multiple of 16"),
    (dict(key_cache=torch.zeros(1, 2, 16, 32).half().expand(4, 2, 16, 32)), ValueError, "expanded"),
    (dict(key_cache=_SAME, value_cache=_SAME), ValueError, "different tensors"),
    (dict(key_cache=torch.zeros(4, 2, 16, 32).half().requires_grad_()), RuntimeError, "no gradients"),
    (dict(sources=[0]), TypeError, "sources"),
    (dict(sources=torch.zeros(1).long()), ValueError, "sources must be int32"),
    (dict(targets=torch.zeros(2).int()), ValueError, "targets must have shape"),
    (dict(tokens=torch.zeros(2).int()), ValueError, "tokens must have shape"),
    (dict(tokens=3), TypeError, "tokens"),
    (dict(backend="triton"), RuntimeError, "CUDA tensor"),
])
def test_copy_refusals(change, error, message):
    with pytest.raises(error, match=message):
        paged_cache_copy(**{**_copy_args(), **change})


@pytest.mark.gpu
def test_copy_kernel_refuses_caches_it_cannot_address():
    a = _copy_args("cuda")
    with pytest.raises(RuntimeError, match="same strides"):
        paged_cache_copy(**{**a, "key_cache": torch.zeros(4, 16, 2, 32, device="cuda").half()
                            .transpose(1, 2)}, backend="triton")
    with pytest.raises(RuntimeError, match="float16 and bfloat16"):
        paged_cache_copy(**_copy_args("cuda", torch.float32), backend="triton")


# ---- compact ----------------------------------------------------------------------------


def check_compact(pages, free, *, B=3, M=4, start=None, seed=0, device="cpu", backend="torch",
                  pad_columns=0):
    rng = random.Random(seed)
    s = min(max(start or 0, 0), len(free))
    gone = {p for p in free[s:] if 0 <= p < pages}
    used = pages - len(gone)
    moves = list(zip([p for p in range(used, pages) if p not in gone],
                     [p for p in range(used) if p in gone]))
    shares = [0 if p in gone else rng.randint(0, 5) for p in range(pages)]
    table = [[rng.choice([-1, rng.randrange(pages), pages + 3]) for _ in range(M)] for _ in range(B)]
    place = dict(moves)
    want_shares = [n if p < used else 0 for p, n in enumerate(shares)]
    for a, b in moves:
        want_shares[b] = shares[a]
    pad = [-1] * (len(free) - len(moves))
    tail = list(range(used, pages))[:len(free) - s]
    t = torch.full((B, M + pad_columns), -9, dtype=torch.int32, device=device)[:, :M]
    if B:
        t.copy_(ints(table, device))
    inputs = [t, ints(free, device), ints(shares, device)]
    kept = [x.clone() for x in inputs]
    c = paged_cache_compact(*inputs, free_start=None if start is None else ints([start], device),
                            backend=backend)
    assert all(torch.equal(a, b) for a, b in zip(inputs, kept))
    assert all(x.dtype == torch.int32 for x in c)
    assert c.used.tolist() == [used] and c.page_shares.tolist() == want_shares
    assert c.page_table.tolist() == [[place.get(p, p) for p in row] for row in table]
    assert c.sources.tolist() == [a for a, _ in moves] + pad
    assert c.targets.tolist() == [b for _, b in moves] + pad
    assert c.free_pages.tolist() == free[:s] + tail + [-1] * (len(free) - s - len(tail))


def some_pages(n, k, seed):
    return random.Random(seed).sample(range(n), k)


COMPACTS = [
    dict(pages=1, free=[]),
    dict(pages=1, free=[0]),
    dict(pages=8, free=[0, 1, 2]),
    dict(pages=8, free=[7, 6]),
    dict(pages=40, free=some_pages(40, 17, 1)),
    dict(pages=64, free=some_pages(64, 60, 2), start=3),
    dict(pages=33, free=list(range(33))),
    dict(pages=70, free=[3, 3, 90, -1, 5, 69], start=0),       # twice, and no pages
    dict(pages=70, free=some_pages(70, 20, 3), start=100),
    dict(pages=70, free=some_pages(70, 20, 3), start=-5),
    dict(pages=9, free=[4], B=0),
]


@pytest.mark.parametrize("case", COMPACTS)
def test_compact_torch_form(case):
    check_compact(**case)


@pytest.mark.gpu
@pytest.mark.parametrize("case", COMPACTS + [
    dict(pages=5000, free=some_pages(5000, 1234, 4), B=50, M=70, pad_columns=5),
    dict(pages=8192, free=some_pages(8192, 8000, 5), B=70, M=33),
    dict(pages=8193, free=some_pages(8193, 100, 6), B=700, M=3),
    dict(pages=100001, free=some_pages(100001, 50000, 7), B=300, M=200, start=11),
    dict(pages=300000, free=some_pages(300000, 290000, 8), B=5, M=100),
])
def test_compact_kernel(case):
    check_compact(**case, device="cuda", backend="triton")


@pytest.mark.gpu
def test_compact_kernel_reads_strided_inputs():
    table = ints([[1, 5], [6, 2], [0, 7]], "cuda").t()
    free, shares = (torch.stack([ints(v, "cuda")] * 2, 1)[:, 0]
                    for v in ([3, 4, 0], [9, 1, 2, 9, 9, 3, 4, 5]))
    got = [paged_cache_compact(table, free, shares, backend=b) for b in ("triton", "torch")]
    assert all(torch.equal(a, b) for a, b in zip(*got))


def _compact_args():
    i = torch.int32
    return dict(page_table=torch.zeros(2, 4, dtype=i), free_pages=torch.arange(8, dtype=i),
                page_shares=torch.zeros(9, dtype=i))


@pytest.mark.parametrize(("change", "error", "message"), [
    (dict(backend="x"), ValueError, "backend"),
    (dict(page_table=torch.zeros(2, 4)), ValueError, "page_table must be int32"),
    (dict(page_table=torch.zeros(4).int()), ValueError, "page_table must have shape"),
    (dict(free_pages=torch.zeros(2).long()), ValueError, "free_pages must be int32"),
    (dict(page_shares=torch.zeros(2, 2).int()), ValueError, "page_shares must have shape"),
    (dict(page_shares=torch.zeros(0).int()), ValueError, "at least one page"),
    (dict(free_start=torch.zeros(1).long()), ValueError, "free_start"),
    (dict(backend="triton"), RuntimeError, "CUDA tensor"),
])
def test_compact_refusals(change, error, message):
    with pytest.raises(error, match=message):
        paged_cache_compact(**{**_compact_args(), **change})


# ---- together ---------------------------------------------------------------------------


class Beams:
    """Beam decoding: two requests of ``K`` beams over prompts that each begins alone. A step's
    keys, values and queries are random; which beams survive is too."""

    S, H, Hq, D, M, K = 16, 2, 4, 32, 10, 3

    def __init__(self, device, backend, dtype, seed):
        self.rng, self.device, self.backend = random.Random(seed), device, backend
        self.gen = torch.Generator().manual_seed(seed)
        B, P = 2 * self.K, 60
        self.B, self.dtype = B, dtype
        self.table, self.lengths = ints([[-1] * self.M] * B, device), ints([0] * B, device)
        self.free, self.shares = ints(list(range(P)), device), ints([0] * P, device)
        self.start = ints([0], device)
        self.caches = [torch.full((P, self.H, self.S, self.D), math.nan, dtype=dtype, device=device)
                       for _ in range(2)]
        self.dense = [[torch.zeros(0, self.H, self.D, dtype=torch.float64)] * 2 for _ in range(B)]
        self.starts = ints([0, self.K, B], device)

    def randn(self, *shape):
        return torch.randn(shape, generator=self.gen).to(self.dtype)

    def append(self, new):
        """New tokens of every sequence into the cache."""
        T = sum(new)
        k, v = self.randn(T, self.H, self.D), self.randn(T, self.H, self.D)
        plan = paged_cache_plan(self.table, self.lengths, ints(new, self.device), self.free,
                                page_size=self.S, num_tokens=T, free_start=self.start,
                                backend=self.backend)
        paged_cache_store(k.to(self.device), v.to(self.device), *self.caches, plan.slots,
                          backend=self.backend)
        self.lengths, self.start = plan.lengths, plan.free_start
        at = 0
        for b, n in enumerate(new):
            self.dense[b] = [torch.cat((d, t[at:at + n].double())) for d, t in zip(self.dense[b], (k, v))]
            at += n

    def fork(self, parents):
        fork = paged_cache_fork(self.table, self.lengths, ints(parents, self.device), self.free,
                                self.shares, page_size=self.S, free_start=self.start,
                                backend=self.backend)
        paged_cache_copy(*self.caches, fork.sources, fork.targets, tokens=fork.tokens,
                         backend=self.backend)
        self.lengths, self.start = fork.lengths, fork.free_start
        self.dense = [self.dense[p] for p in parents]

    def compact(self):
        c = paged_cache_compact(self.table, self.free, self.shares, free_start=self.start,
                                backend=self.backend)
        paged_cache_copy(*self.caches, c.sources, c.targets, backend=self.backend)
        self.table, self.free, self.shares = c.page_table, c.free_pages, c.page_shares

    def attend(self):
        """Pages that a group's rows have in common are its prefix."""
        table, lens = self.table.tolist(), self.lengths.tolist()
        prefix = []
        for g in range(2):
            rows = range(g * self.K, (g + 1) * self.K)
            same = 0
            while all(same < lens[b] // self.S and table[b][same] == table[rows[0]][same] for b in rows):
                same += 1
            prefix.append(same * self.S)
        q = self.randn(self.B, self.Hq, 1, self.D)
        o = paged_prefix_attention(q.to(self.device), *self.caches, self.table, self.lengths,
                                   self.starts, ints(prefix, self.device), enable_gqa=True,
                                   backend=self.backend)
        want, bound = attention_reference(q, self.dense, self.D ** -0.5, self.dtype)
        within(o, want, bound, self.dtype)
        return prefix


def decode(device, backend, dtype, seed):
    d = Beams(device, backend, dtype, seed)
    prompts = [d.rng.randint(20, 60) for _ in range(2)]
    d.append([prompts[b // d.K] if b % d.K == 0 else 0 for b in range(d.B)])
    d.fork([b // d.K * d.K for b in range(d.B)])
    shared = 0
    for step in range(30):
        d.append([1] * d.B)
        shared += sum(d.attend())
        d.fork([b // d.K * d.K + d.rng.randrange(d.K) for b in range(d.B)])
        if step % 10 == 9:
            d.compact()
    assert shared > 0
    held = {p for row, n in zip(d.table.tolist(), d.lengths.tolist()) for p in row[:cdiv(n, d.S)]}
    assert int(d.start) == len(held)


@pytest.mark.parametrize("seed", range(2))
def test_beam_decoding_torch_form(seed):
    decode("cpu", "torch", torch.float32, seed)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("seed", range(3))
def test_beam_decoding_kernels(seed, dtype):
    decode("cuda", "triton", dtype, seed)
