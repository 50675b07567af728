"""How the operators on shared pages are called: batches past what a work-group keeps in LDS, strided
arguments, the C++ binding and the op layer, other streams, threads, captured steps, torch.compile
and gradients."""

from __future__ import annotations

import random
import threading

import pytest
import torch
from test_paged import attention_reference, cdiv
from test_pages import (Beams, check_compact, check_copy, check_fork, decode, ints, some_pages,
                        some_parents)
from test_prefix import check_prefix, make_shared, many, within

from triton_flash_attention import (_native, paged_cache_compact, paged_cache_copy, paged_cache_fork,
                                    paged_cache_plan, paged_cache_store, paged_prefix_attention)

# More sequences than 2048, or groups than 1023: starts, prefixes and lengths are read from memory.
BEYOND = [
    (*many([2] * 1040 + [1] * 3 + [17], 1, 40, 1), 2, 1, 1, 32, 16),
    (*many([2100], 100, 100, 2), 2, 1, 1, 64, 16),
    (*many([1] * 1030 + [2] * 30, 1, 60, 3), 2, 2, 1, 32, 16),
    (*many([700, 1, 1400], 16, 90, 4), 2, 1, 33, 32, 16),
    (*many([1] * 1100 + [3] * 10, 1, 60, 5), 4, 1, 17, 128, 16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", BEYOND)
def test_prefix_kernel_of_more_than_a_work_group_keeps(case):
    check_prefix(*case, torch.float16, device="cuda", backend="triton")


@pytest.mark.gpu
def test_prefix_kernel_where_the_grid_leaves_no_room_for_pieces():
    """Nine tiles that meet long prefixes, 12 units of 32 keys each, beside own keys of 5953 units: the
    line's stretches are of 12, 497 work-groups of 512 go to own keys, and the nine pieces, which come
    in eights, stay on the line."""
    check_prefix([3, 3, 3], [384] * 3, [384] * 9 + [94 * 32] * 59 + [47 * 32], 4, 1, 25, 128, 32,
                 torch.bfloat16, device="cuda", backend="triton")


def spread(t):
    """The same values behind a stride of two elements."""
    wide = torch.full((*t.shape[:-1], 2 * t.shape[-1]), -77, dtype=t.dtype, device=t.device)
    wide[..., ::2] = t
    return wide[..., ::2]


def strided_calls(device, backend, dtype):
    sizes, prefix, lengths = [3, 1, 2], [20, 4, 33], [40, 21, 25, 9, 50, 37]
    views, table, starts, dense = make_shared(sizes, prefix, lengths, 2, 16, 64, dtype, device=device)
    q = torch.randn(6, 4, 1, 64, generator=torch.Generator().manual_seed(3)).to(dtype)
    o = paged_prefix_attention(q.to(device), *views, spread(table), spread(ints(lengths, device)),
                               spread(starts), spread(ints(prefix, device)), enable_gqa=True,
                               backend=backend)
    within(o, *attention_reference(q, dense, 64 ** -0.5, dtype), dtype)
    caches = [torch.randn(7, 2, 16, 32, device=device).to(dtype) for _ in range(2)]
    want = [c.clone() for c in caches]
    for w in want:
        w[0, :, :5], w[6] = w[2, :, :5], w[4]
    paged_cache_copy(*caches, *(spread(ints(v, device)) for v in ([2, 4], [0, 6])),
                     tokens=spread(ints([5, 16], device)), backend=backend)
    assert all(torch.equal(c, w) for c, w in zip(caches, want))
    t = ints([[0, 1], [-1, -1]], device)
    f = paged_cache_fork(t, spread(ints([20, 0], device)), spread(ints([0, 0], device)),
                         ints([2, 3], device), ints([0] * 4, device), page_size=16, backend=backend)
    assert t.tolist() == [[0, 1], [0, 2]] and f.targets.tolist() == [-1, 2]


def test_strided_arguments_torch_forms():
    strided_calls("cpu", "torch", torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_strided_arguments_kernels(native, monkeypatch):
    if not native:
        monkeypatch.setattr(_native, "available", lambda: False)
    strided_calls("cuda", "triton", torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_binding_and_op_layer(native, monkeypatch):
    """The same calls through the C++ binding and without it."""
    assert _native.available(), _native.status()[1]
    if not native:
        monkeypatch.setattr(_native, "available", lambda: False)
    check_prefix([3, 1, 0, 2], [130, 16, 9, 300], [150, 131, 200, 40, 310, 305, 20], 8, 2, 3, 96, 48,
                 torch.bfloat16, layout="tokens", q_layout="tokens", device="cuda", backend="triton")
    for S, pad in ((16, 0), (48, 3)):
        check_fork([20, 30, 40, 50, 0], some_parents(5, S), S, pad_columns=pad, device="cuda",
                   backend="triton")
    for part in (False, True):
        check_copy(26, 60, 5, 80, 16, torch.float16, layout="tokens", part=part, device="cuda",
                   backend="triton")
    check_compact(pages=500, free=some_pages(500, 200, 1), B=9, M=30, start=5, pad_columns=1,
                  device="cuda", backend="triton")
    decode("cuda", "triton", torch.float16, 5)


@pytest.mark.gpu
def test_kernels_from_two_threads_on_two_streams():
    """Calls at once, each with tensors and a workspace of its own."""
    failures = []

    def work(seed):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for i in range(3):
                    check_prefix(*many([5, 1, 3], 1, 900, 10 * seed + i), 8, 2, 1, 64, 16,
                                 torch.float16, seed=i, device="cuda", backend="triton")
                    check_fork([100] * 40, some_parents(40, seed + i), 16, device="cuda",
                               backend="triton")
                    check_compact(pages=9000 * seed + 500, free=some_pages(500, 200, i), B=9, M=30,
                                  device="cuda", backend="triton")
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
def test_kernels_on_another_stream():
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        decode("cuda", "triton", torch.bfloat16, 6)
    side.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("pages", [60, 20000])
def test_beam_step_captured_and_replayed(pages):
    """A whole step of beam search in a graph, with as many pages as small calls take and more; every
    replay against the same step run eagerly on copies, and the attention against 64 bits."""
    d = Beams("cuda", "triton", torch.float16, 7)
    d.free, d.shares = ints(list(range(pages)), "cuda"), ints([0] * pages, "cuda")
    d.caches = [torch.zeros(pages, d.H, d.S, d.D, dtype=d.dtype, device="cuda") for _ in range(2)]
    d.append([37 if b % d.K == 0 else 0 for b in range(d.B)])
    d.fork([b // d.K * d.K for b in range(d.B)])
    z = dict(dtype=d.dtype, device="cuda")
    k, v = (torch.zeros(d.B, d.H, d.D, **z) for _ in range(2))
    q = torch.zeros(d.B, d.Hq, 1, d.D, **z)
    one, parents, prefix = ints([1] * d.B, "cuda"), ints([0] * d.B, "cuda"), ints([0, 0], "cuda")

    def step(table, lengths, free, shares, start, kc, vc):
        plan = paged_cache_plan(table, lengths, one, free, page_size=d.S, num_tokens=d.B,
                                free_start=start, backend="triton")
        paged_cache_store(k, v, kc, vc, plan.slots, backend="triton")
        o = paged_prefix_attention(q, kc, vc, table, plan.lengths, d.starts, prefix, enable_gqa=True,
                                   backend="triton")
        fork = paged_cache_fork(table, plan.lengths, parents, free, shares, page_size=d.S,
                                free_start=plan.free_start, backend="triton")
        paged_cache_copy(kc, vc, fork.sources, fork.targets, tokens=fork.tokens, backend="triton")
        c = paged_cache_compact(table, free, shares, free_start=fork.free_start, backend="triton")
        paged_cache_copy(kc, vc, c.sources, c.targets, backend="triton")
        for a, b in ((table, c.page_table), (free, c.free_pages), (shares, c.page_shares),
                     (lengths, fork.lengths), (start, fork.free_start)):
            a.copy_(b)
        return o

    state = [d.table, d.lengths.clone(), d.free, d.shares, d.start.clone(), *d.caches]
    step(*(t.clone() for t in state))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*state)
    rng = random.Random(3)
    shared = 0
    for i in range(24):
        for t in (k, v, q):
            t.copy_(d.randn(*t.shape))
        table, lens = state[0].tolist(), state[1].tolist()
        same = []
        for g in range(2):
            rows = range(g * d.K, (g + 1) * d.K)
            n = 0
            while all(n < lens[b] // d.S and table[b][n] == table[rows[0]][n] for b in rows):
                n += 1
            same.append(n * d.S)
        shared += sum(same)
        prefix.copy_(ints(same))
        chosen = [b // d.K * d.K + rng.randrange(d.K) for b in range(d.B)]
        parents.copy_(ints(chosen))
        eager = [t.clone() for t in state]
        want = step(*eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        assert all(torch.equal(a, b) for a, b in zip(state, eager)), i
        d.dense = [[torch.cat((x, t[b:b + 1].double().cpu())) for x, t in zip(d.dense[b], (k, v))]
                   for b in range(d.B)]
        within(out, *attention_reference(q, d.dense, d.D ** -0.5, d.dtype), d.dtype)
        d.dense = [d.dense[p] for p in chosen]
    held = {p for row, n in zip(state[0].tolist(), state[1].tolist()) for p in row[:cdiv(n, d.S)]}
    assert shared > 0 and held == set(range(int(state[4])))


@pytest.mark.gpu
def test_two_captured_calls_replayed_in_turn():
    """Two graphs that share torch's pool: each keeps its own partials."""
    cases = [make_shared([3, 2], [900, 40], [1000, 950, 930, 60, 700], 2, 16, 64, torch.float16,
                         device="cuda", seed=s) for s in (1, 2)]
    lens, prefix = ints([1000, 950, 930, 60, 700], "cuda"), ints([900, 40], "cuda")
    gen = torch.Generator().manual_seed(4)
    q = torch.randn(5, 8, 1, 64, generator=gen).half().cuda()

    def call(views, table, starts, dense):
        return paged_prefix_attention(q, *views, table, lens, starts, prefix, enable_gqa=True,
                                      backend="triton")

    pool = torch.cuda.graph_pool_handle()
    graphs, outs = [], []
    for case in cases:
        call(*case)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(call(*case))
        graphs.append(g)
    for i in range(3):
        q.copy_(torch.randn(5, 8, 1, 64, generator=gen).half())
        wants = [call(*case) for case in cases]
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, wants)), i


def compiled(device, dtype, **kwargs):
    views, table, starts, _ = make_shared([2], [20], [40, 33, 9], 2, 16, 32, dtype, device=device, fill=0.0)
    q = torch.randn(3, 4, 1, 32, generator=torch.Generator().manual_seed(1)).to(dtype).to(device)
    lens, prefix, parents = ints([40, 33, 9], device), ints([20], device), ints([1, 1, 0], device)
    pages = views[0].shape[0]

    def f(q, table, free, shares, kc, vc):
        o = paged_prefix_attention(q * 2, kc, vc, table, lens, starts, prefix, enable_gqa=True)
        fork = paged_cache_fork(table, lens, parents, free, shares, page_size=16)
        paged_cache_copy(kc, vc, fork.sources, fork.targets, tokens=fork.tokens)
        return o + 1, fork.lengths, fork.targets, fork.free_start

    runs = []
    torch._dynamo.reset()
    for run in (f, torch.compile(f, backend="eager", **kwargs)):
        state = [table.clone(), ints(list(range(pages)), device), ints([1] * pages, device),
                 *(v.clone() for v in views)]
        with torch.no_grad():
            runs.append([*run(q, *state), *state])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_torch_forms_compile():
    compiled("cpu", torch.float32)


@pytest.mark.gpu
def test_kernels_under_torch_compile():
    """Calls that the kernels serve run beside the compiled graph, with the same results."""
    compiled("cuda", torch.float16)


def attend(q, views, table, starts, backend="auto"):
    return paged_prefix_attention(q, *views, table, ints([40, 33, 9], q.device), starts,
                                  ints([20], q.device), enable_gqa=True, backend=backend)


def test_torch_form_has_gradients():
    """Against differences, of a query, and of a prefix's keys and values, which all rows share."""
    views, table, starts, _ = make_shared([2], [20], [40, 33, 9], 2, 16, 8, torch.float64, fill=0.0)
    gen = torch.Generator().manual_seed(2)
    q = torch.randn(3, 4, 1, 8, generator=gen, dtype=torch.float64)
    w = torch.randn(3, 4, 1, 8, generator=gen, dtype=torch.float64)
    leaves = [t.clone().requires_grad_() for t in (q, *views)]
    (attend(leaves[0], leaves[1:], table, starts) * w).sum().backward()
    for n, x in enumerate(leaves):
        along = torch.randn(x.shape, generator=gen, dtype=torch.float64)
        step = 1e-5
        ends = []
        for s in (step, -step):
            moved = [t.detach() + s * along if i == n else t.detach() for i, t in enumerate(leaves)]
            ends.append((attend(moved[0], moved[1:], table, starts) * w).sum())
        want = (ends[0] - ends[1]) / (2 * step)
        # central differences: 1e-10 of the third derivative, and 2^-52 / 1e-5 of the sum
        assert torch.allclose((x.grad * along).sum(), want, rtol=1e-7, atol=1e-7)


@pytest.mark.gpu
def test_kernels_record_no_gradients():
    views, table, starts, _ = make_shared([2], [20], [40, 33, 9], 2, 16, 32, torch.float16, fill=0.0,
                                          device="cuda")
    q = torch.randn(3, 4, 1, 32, device="cuda").half().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        attend(q, views, table, starts, backend="triton")
    attend(q, views, table, starts).sum().backward()  # in PyTorch
    assert q.grad.isfinite().all() and bool(q.grad.any())
    with torch.no_grad():
        attend(q, views, table, starts, backend="triton")
    caches = [v.clone().requires_grad_() for v in views]
    for backend in ("auto", "triton", "torch"):
        with pytest.raises(RuntimeError, match="records no gradients"):
            paged_cache_copy(*caches, ints([0], "cuda"), ints([1], "cuda"), backend=backend)


@pytest.mark.gpu
def test_inputs_stay_as_they_are():
    """What the attention reads and what a fork only reads, and the workspaces' neighbours."""
    views, table, starts, _ = make_shared([2], [20], [40, 33, 9], 2, 16, 32, torch.float16, fill=0.0,
                                          device="cuda")
    q = torch.randn(3, 4, 1, 32, device="cuda").half()
    lens, parents = ints([40, 33, 9], "cuda"), ints([2, 0, 0], "cuda")
    kept = [t.clone() for t in (q, *views, table, starts, lens, parents)]
    attend(q, views, table, starts, backend="triton")
    pages = views[0].shape[0]
    paged_cache_fork(table.clone(), lens, parents, ints(list(range(pages)), "cuda"),
                     ints([1] * pages, "cuda"), page_size=16, backend="triton")
    assert all(torch.equal(a, b) for a, b in zip(kept, (q, *views, table, starts, lens, parents)))
