"""qk_norm_rope against its formulas in 64 bits: the PyTorch form on the CPU, the gfx950
kernels on the GPU (forward, backward, strides, positions, refusals).

Tolerances, element by element. An output is rounded once to its type, by at most half a step:
``u = finfo(type).eps / 2`` relative (fp16 below 2^-14: 2^-25 absolute). Before that it is the
result of some 30 float32 operations on values no larger than the row's largest (a sum of at
most 128 squares in a tree of depth below 16, a reciprocal root of 1 ulp, two products, a
rotation): below 64 units of 2^-24 of the row's largest summand. The backward's rows chain two
such sums: 256 units. A weight's gradient adds n products in float32, each off by at most 32
units, in any order: at most (n + 32) 2^-24 of the sum of their magnitudes."""

from __future__ import annotations

import math

import pytest
import torch

from triton_flash_attention import _native, qk_norm_rope

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
F32 = 2.0 ** -24


def tables(P, R, device="cpu", base=10000.0):
    angle = torch.arange(P, dtype=torch.float64)[:, None] * base ** (
        -torch.arange(0, R, 2, dtype=torch.float64) / R)
    return angle.cos().float().to(device), angle.sin().float().to(device)


def pair_index(R, interleaved):
    i = torch.arange(R // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)


def turn(y, cos, sin, interleaved, direction):
    R = 2 * cos.shape[-1]
    a, b = pair_index(R, interleaved)
    z = y.clone()
    z[..., a] = y[..., a] * cos - direction * y[..., b] * sin
    z[..., b] = y[..., b] * cos + direction * y[..., a] * sin
    return z


def reference(x, w, cos, sin, eps, positions, interleaved, g=None):
    """(z, its bound, dx, its bound, dw, its bound) in float64, for one tensor on the CPU."""
    B, H, N, D = x.shape
    x = x.double()
    pos = torch.arange(N) if positions is None else positions.long()
    pos = pos.expand(B, N)
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    r = torch.ones(B, H, N, 1, dtype=torch.float64)
    ww = torch.ones(D, dtype=torch.float64)
    if w is not None:
        ww = w.double()
        r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    unit = x * r
    y = unit * ww
    z = turn(y, c, s, interleaved, 1)
    z_bound = 64 * F32 * y.abs().amax(-1, keepdim=True)
    if g is None:
        return z, z_bound
    u = turn(g.double(), c, s, interleaved, -1)
    if w is None:
        return z, z_bound, u, 64 * F32 * g.double().abs().amax(-1, keepdim=True)
    t = u * ww
    mean = (t * unit).mean(-1, keepdim=True)
    mean_abs = (t * unit).abs().mean(-1, keepdim=True)
    dx = r * (t - unit * mean)
    dx_bound = 256 * F32 * (r * (t.abs() + unit.abs() * mean_abs)).amax(-1, keepdim=True)
    terms = u * unit
    # u itself is off by a few units of its pair's larger value
    size = (g.double().abs().amax(-1, keepdim=True) * unit.abs())
    return (z, z_bound, dx, dx_bound, terms.sum((0, 1, 2)),
            (B * H * N + 32) * F32 * size.sum((0, 1, 2)))


def close(name, got, want, bound, dtype):
    got = got.detach().double().cpu()
    limit = HALF[dtype] * want.abs() * 1.0001 + bound + 2.0 ** -25
    off = (got - want).abs()
    worst = (off / limit).max().item()
    assert got.shape == want.shape and bool((off <= limit).all()), f"{name}: {worst:.3f} of the bound"


def inputs(B, Hq, Hkv, N, D, dtype, seed, layout="heads", device="cpu"):
    gen = torch.Generator().manual_seed(seed)
    if layout == "heads":
        q, k = (torch.randn(B, H, N, D, generator=gen).to(dtype).to(device) for H in (Hq, Hkv))
    else:  # slices of a fused projection
        f = torch.randn(B, N, Hq + Hkv, D, generator=gen).to(dtype).to(device)
        q, k = f[:, :, :Hq].transpose(1, 2), f[:, :, Hq:].transpose(1, 2)
    gq, gk = (torch.randn(B, H, N, D, generator=gen).to(dtype).to(device) for H in (Hq, Hkv))
    wq, wk = (1 + 0.3 * torch.randn(D, generator=gen) for _ in range(2))
    return q, k, gq, gk, wq, wk


def check(B, Hq, Hkv, N, D, R, dtype, *, norm=True, interleaved=False, layout="heads",
          positions=None, P=None, w_dtype=None, device="cpu", backend="torch", seed=0, train=True):
    q, k, gq, gk, wq, wk = inputs(B, Hq, Hkv, N, D, dtype, seed, layout, device)
    w_dtype = w_dtype or dtype
    wq, wk = ((wq.to(w_dtype).to(device), wk.to(w_dtype).to(device)) if norm else (None, None))
    cos, sin = tables(P or N, R, device)
    pos = None if positions is None else positions.to(device)
    leaves = [q, k] + ([wq, wk] if norm else [])
    if train:
        leaves = [t.detach().requires_grad_() for t in leaves]
    args = dict(eps=1e-6, positions=pos, interleaved=interleaved, backend=backend)
    if norm:
        args.update(query_weight=leaves[2], key_weight=leaves[3])
    oq, ok = qk_norm_rope(leaves[0], leaves[1], cos, sin, **args)
    assert oq.is_contiguous() and ok.is_contiguous() and oq.dtype == dtype
    grads = torch.autograd.grad((oq, ok), leaves, (gq, gk)) if train else None
    for i, (n, x, w, o, g) in enumerate((("query", q, wq, oq, gq), ("key", k, wk, ok, gk))):
        ref = reference(x.cpu(), None if w is None else w.cpu(), cos.cpu(), sin.cpu(), 1e-6,
                        positions, interleaved, g.cpu() if train else None)
        close(n, o, ref[0], ref[1], dtype)
        if train:
            close("d" + n, grads[i], ref[2], ref[3], dtype)
            if norm:
                close("dw " + n, grads[2 + i], ref[4], ref[5], w_dtype)


def positions_of(kind, B, N, P, seed=5):
    gen = torch.Generator().manual_seed(seed)
    if kind == "none":
        return None
    if kind == "shared":  # [N], int64, in any order, with repeats
        return torch.randint(0, P, (N,), generator=gen)
    return torch.randint(0, P, (B, N), generator=gen).int()


# (B, Hq, Hkv, N, D, R, norm, interleaved, layout, positions)
SHAPES = [
    (1, 1, 1, 1, 16, 16, True, False, "heads", "none"),
    (2, 4, 2, 5, 64, 64, True, False, "tokens", "each"),
    (1, 3, 1, 7, 128, 128, True, True, "tokens", "shared"),
    (2, 2, 2, 9, 80, 32, True, False, "heads", "each"),
    (1, 2, 1, 33, 40, 16, True, True, "heads", "none"),
    (2, 8, 2, 1, 128, 64, False, False, "tokens", "each"),
    (1, 2, 2, 17, 32, 32, False, True, "heads", "shared"),
    (1, 5, 1, 3, 72, 48, True, False, "heads", "none"),
    (3, 2, 1, 11, 8 * 13, 96, False, False, "heads", "each"),
]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_torch_form(shape, dtype):
    B, Hq, Hkv, N, D, R, norm, inter, layout, pos = shape
    check(B, Hq, Hkv, N, D, R, dtype, norm=norm, interleaved=inter, layout=layout,
          positions=positions_of(pos, B, N, 50), P=50)


def test_torch_form_serves_what_the_kernels_do_not():
    check(1, 2, 1, 4, 12, 10, torch.float32)
    check(1, 2, 1, 4, 256, 2, torch.float16, interleaved=True)


def test_gradients_against_differences():
    gen = torch.Generator().manual_seed(3)
    q, k = (torch.randn(1, h, 3, 8, generator=gen, dtype=torch.float64, requires_grad=True)
            for h in (2, 1))
    wq, wk = (torch.rand(8, generator=gen, dtype=torch.float64).add(0.5).requires_grad_()
              for _ in range(2))
    cos, sin = tables(9, 6)
    pos = torch.tensor([[8, 0, 8]])
    for inter in (False, True):
        assert torch.autograd.gradcheck(
            lambda *t: qk_norm_rope(t[0], t[1], cos, sin, query_weight=t[2], key_weight=t[3],
                                    positions=pos, interleaved=inter), (q, k, wq, wk))


def test_eps_of_any_real_type():
    from fractions import Fraction

    q, w = torch.randn(1, 2, 3, 16), torch.ones(16)
    args = (q, q, *tables(3, 8))
    want = qk_norm_rope(*args, query_weight=w, key_weight=w, eps=0.5)[0]
    assert torch.equal(qk_norm_rope(*args, query_weight=w, key_weight=w, eps=Fraction(1, 2))[0], want)
    assert not qk_norm_rope(*args, query_weight=w, key_weight=w, eps=10 ** 40)[0].any()


def test_positions_outside_the_tables_are_nan():
    q, k = torch.randn(1, 2, 3, 16), torch.randn(1, 1, 3, 16)
    cos, sin = tables(4, 8)
    for bad in (-1, 4, 1 << 30):
        oq, ok = qk_norm_rope(q, k, cos, sin, positions=torch.tensor([0, bad, 3]))
        for o in (oq, ok):
            assert o[:, :, 1].isnan().all() and not o[:, :, 0::2].isnan().any()


def check_gradients_of_bad_positions(norm, interleaved, each, device, backend, dtype):
    """Tokens outside the tables have NaN for their gradients, and so have the weights; the other
    tokens' gradients are those of a call without them."""
    B, N, D, R = 2, 5, 48, 32
    q, k, gq, gk, wq, wk = inputs(B, 4, 2, N, D, dtype, 7, device=device)
    cos, sin = tables(6, R, device)
    if each:
        pos = torch.tensor([[0, 1, 2, 3, 6], [-1, 5, 4, 1 << 30, 0]], device=device)
    else:
        pos = torch.tensor([3, -7, 5, 6, 0], device=device)
    bad = ((pos < 0) | (pos >= 6)).expand(B, N)

    def grads(positions):
        leaves = [t.detach().requires_grad_() for t in (q, k)]
        weights = {}
        if norm:
            leaves += [w.to(device).requires_grad_() for w in (wq, wk)]
            weights = dict(query_weight=leaves[2], key_weight=leaves[3])
        out = qk_norm_rope(leaves[0], leaves[1], cos, sin, positions=positions,
                           interleaved=interleaved, backend=backend, **weights)
        return torch.autograd.grad(out, leaves, (gq, gk))

    got, want = grads(pos), grads(torch.where((pos < 0) | (pos >= 6), 0, pos))
    for g, w in zip(got[:2], want):
        rows = bad[:, None, :, None].expand_as(g)
        assert g[rows].isnan().all() and torch.equal(g[~rows], w[~rows])
    assert all(g.isnan().all() for g in got[2:]) and not any(w.isnan().any() for w in want)


BAD_POSITIONS = [(n, i, e) for n in (True, False) for i in (True, False) for e in (True, False)]


@pytest.mark.parametrize(("norm", "interleaved", "each"), BAD_POSITIONS)
def test_gradients_of_positions_outside_the_tables(norm, interleaved, each):
    for dtype in (torch.float32, torch.float64, torch.bfloat16):
        check_gradients_of_bad_positions(norm, interleaved, each, "cpu", "torch", dtype)


@pytest.mark.gpu
@pytest.mark.parametrize(("norm", "interleaved", "each"), BAD_POSITIONS)
def test_kernel_gradients_of_positions_outside_the_tables(norm, interleaved, each):
    for dtype in (torch.float16, torch.bfloat16):
        check_gradients_of_bad_positions(norm, interleaved, each, "cuda", "triton", dtype)


def test_tables_take_no_gradient_from_positions_outside_them():
    q = torch.randn(1, 2, 3, 16)
    leaves = [t.requires_grad_() for t in tables(4, 8)]
    out = qk_norm_rope(q, q, *leaves, positions=torch.tensor([1, 4, 3]))
    got = torch.autograd.grad(sum(o.sum() for o in out), leaves)
    out = qk_norm_rope(q[:, :, ::2], q[:, :, ::2], *leaves, positions=torch.tensor([1, 3]))
    want = torch.autograd.grad(sum(o.sum() for o in out), leaves)
    assert all(torch.equal(g, w) for g, w in zip(got, want))


def _valid():
    cos, sin = tables(8, 16)
    return dict(query=torch.randn(1, 2, 4, 32), key=torch.randn(1, 1, 4, 32), cos=cos, sin=sin)


@pytest.mark.parametrize(("change", "error", "message"), [
    (dict(backend="cuda"), ValueError, "backend must be one of"),
    (dict(query=[1]), TypeError, "query must be a torch.Tensor"),
    (dict(query=torch.zeros(2, 4, 32)), ValueError, "query must have shape"),
    (dict(key=torch.zeros(1, 0, 4, 32)), ValueError, "greater than zero"),
    (dict(query=torch.zeros(1, 2, 4, 32, dtype=torch.int32)), ValueError, "floating-point"),
    (dict(key=torch.zeros(1, 1, 4, 32, dtype=torch.float16)), ValueError, "same dtype"),
    (dict(key=torch.zeros(1, 1, 5, 32)), ValueError, "must match"),
    (dict(cos=torch.zeros(8, 8, dtype=torch.float16)), ValueError, "cos must be float32"),
    (dict(cos=torch.zeros(8, 7)), ValueError, "same shape"),
    (dict(cos=torch.zeros(8, 17), sin=torch.zeros(8, 17)), ValueError, "head_dim / 2"),
    (dict(query_weight=torch.ones(32)), ValueError, "both be given"),
    (dict(query_weight=torch.ones(31), key_weight=torch.ones(31)), ValueError, "head_dim = 32"),
    (dict(query_weight=torch.ones(32).half(), key_weight=torch.ones(32).half()), ValueError,
     "both float32"),
    (dict(eps=-1.0), ValueError, "eps"),
    (dict(eps=float("nan")), ValueError, "eps"),
    (dict(interleaved=1), TypeError, "interleaved"),
    (dict(cos=torch.zeros(3, 8), sin=torch.zeros(3, 8)), ValueError, "3 rows for 4 tokens"),
    (dict(positions=[0, 1, 2, 3]), TypeError, "positions"),
    (dict(positions=torch.zeros(2, 4).long()), ValueError, "positions must have shape"),
    (dict(positions=torch.zeros(4)), ValueError, "int32 or int64"),
])
def test_refusals(change, error, message):
    args = {**_valid(), **change}
    with pytest.raises(error, match=message):
        qk_norm_rope(args.pop("query"), args.pop("key"), args.pop("cos"), args.pop("sin"), **args)


def test_triton_backend_raises_on_the_cpu():
    a = _valid()
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        qk_norm_rope(*a.values(), backend="triton")


# ---- the kernels ------------------------------------------------------------------------

GPU_SHAPES = SHAPES + [
    (2, 32, 8, 129, 128, 128, True, False, "tokens", "none"),
    (1, 16, 16, 515, 64, 32, True, True, "heads", "shared"),
    (4, 8, 8, 1, 96, 96, True, False, "tokens", "each"),
    (1, 40, 8, 1030, 128, 128, False, False, "heads", "none"),
    (1, 3, 2, 2049, 24, 16, True, False, "heads", "none"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", GPU_SHAPES)
def test_kernel(shape, dtype):
    B, Hq, Hkv, N, D, R, norm, inter, layout, pos = shape
    P = max(N, 50)
    check(B, Hq, Hkv, N, D, R, dtype, norm=norm, interleaved=inter, layout=layout,
          positions=positions_of(pos, B, N, P), P=P, device="cuda", backend="triton",
          seed=N + D)


@pytest.mark.gpu
def test_kernel_inference_and_float32_weights():
    check(2, 8, 2, 65, 128, 128, torch.bfloat16, device="cuda", backend="triton", train=False)
    check(2, 8, 2, 65, 128, 128, torch.bfloat16, device="cuda", backend="triton",
          w_dtype=torch.float32)


@pytest.mark.gpu
def test_kernel_and_torch_agree_on_bad_positions_and_infinities():
    gen = torch.Generator().manual_seed(1)
    q, k = (torch.randn(2, h, 5, 64, generator=gen).half().cuda() for h in (4, 2))
    q[0, 1, 2, 40] = math.inf  # behind the rotated values: it reaches only its row's norm
    k[1, 0, 3, 3] = math.nan
    cos, sin = tables(6, 32, "cuda")
    pos = torch.tensor([[0, 1, 2, 3, 6], [-1, 5, 4, 1 << 40, 0]]).cuda()
    w = torch.ones(64, dtype=torch.float16, device="cuda")
    for weights in ({}, dict(query_weight=w, key_weight=w)):
        got, want = (qk_norm_rope(q, k, cos, sin, positions=pos, backend=b, **weights)
                     for b in ("triton", "torch"))
        for g, e in zip(got, want):
            assert torch.equal(g.isnan(), e.isnan()) and torch.equal(g.isinf(), e.isinf())
            assert g[0, :, 4].isnan().all() and g[1, :, 0].isnan().all()


@pytest.mark.gpu
def test_kernel_reads_expanded_and_odd_inputs():
    """A query shared by all heads (a head stride of 0), rows that are not 16-byte aligned,
    tables that are views; gradients of broadcast leaves add up."""
    gen = torch.Generator().manual_seed(2)
    base = torch.randn(2, 1, 6, 64, generator=gen).to(torch.bfloat16).cuda().requires_grad_()
    wide = torch.randn(2, 2, 6, 65, generator=gen).to(torch.bfloat16).cuda()
    k = wide[..., 1:]
    cos, sin = (t[:, ::2] for t in tables(9, 64, "cuda"))
    g = torch.randn(2, 4, 6, 64, generator=gen).to(torch.bfloat16).cuda()
    oq, ok = qk_norm_rope(base.expand(2, 4, 6, 64), k, cos, sin, backend="triton")
    zero = torch.zeros_like(ok)
    (grad,) = torch.autograd.grad((oq, ok), base, (g, zero))
    ref = reference(base.detach().cpu().expand(2, 4, 6, 64), None, cos.cpu(), sin.cpu(), 1e-6, None,
                    False, g.cpu())
    close("query", oq, ref[0], ref[1], torch.bfloat16)
    # torch adds the four heads' gradients, rounded to bf16, and rounds their sum
    limit = HALF[torch.bfloat16] * (ref[2].abs().sum(1, keepdim=True) * 2) + 1e-4
    want = ref[2].sum(1, keepdim=True)
    assert ((grad.double().cpu() - want).abs() <= limit).all()
    close("key", ok, *reference(k.cpu(), None, cos.cpu(), sin.cpu(), 1e-6, None, False),
          torch.bfloat16)


@pytest.mark.gpu
def test_kernel_past_32_bits():
    """Queries of more than 2^32 bytes and 2^31 values, as views of the projection's layout."""
    N, H, D = 460_000, 40, 128
    gen = torch.Generator(device="cuda").manual_seed(1)
    q = torch.empty(1, N, H, D, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    q = q.transpose(1, 2)
    assert q.numel() > 1 << 31
    k = q[:, :1]
    cos, sin = tables(4096, D, "cuda")
    pos = torch.arange(N, device="cuda") % 4096
    oq, ok = qk_norm_rope(q, k, cos, sin, positions=pos, backend="triton")
    for h, n in ((0, 0), (39, N - 5), (20, 233_000)):
        part = q[:, h:h + 1, n:n + 5].cpu()
        ref = reference(part, None, cos.cpu(), sin.cpu(), 1e-6, pos[n:n + 5].cpu(), False)
        close("query", oq[:, h:h + 1, n:n + 5], *ref, torch.bfloat16)
    assert torch.equal(ok, oq[:, :1])


@pytest.mark.gpu
def test_kernel_of_more_tokens_than_a_grid_holds():
    """2^24 blocks of 32 tokens and some: rows 16 bytes apart of one buffer, 77 GB a result."""
    N, D = (1 << 29) + 77, 72
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 180 << 30:
        pytest.skip("needs 180 GB of free GPU memory")
    gen = torch.Generator(device="cuda").manual_seed(1)
    base = torch.empty(8 * N + D, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    q = base.as_strided((1, 1, N, D), (0, 0, 8, 1))
    cos, sin = tables(64, 64, "cuda")
    pos = (torch.arange(N, dtype=torch.int32, device="cuda") % 64)
    oq, ok = qk_norm_rope(q, q, cos, sin, positions=pos, backend="triton")
    edge = (1 << 29) - 32
    for n in (0, 12345, edge - 40, edge, 1 << 29, N - 40):
        part = slice(n, n + 40)
        ref = reference(q[:, :, part].cpu(), None, cos.cpu(), sin.cpu(), 1e-6, pos[part].cpu(), False)
        for o in (oq, ok):
            close("query", o[:, :, part], *ref, torch.bfloat16)
    del oq, ok, o, base, q, pos
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_kernel_norms_of_small_and_large_rows(dtype):
    """Rows whose squares reach both ends of float32's range, and a row of zeros, as PyTorch."""
    scale = [0.0, 6e-8, 1e-4, 1.0, 6e4] if dtype == torch.float16 else [0.0, 1e-18, 1e-4, 1e4, 1e18]
    q = torch.randn(1, 1, 5, 64, generator=torch.Generator().manual_seed(2))
    q = (q.clamp(-1, 1) * torch.tensor(scale)[:, None]).to(dtype).cuda()
    w = torch.ones(64, dtype=dtype, device="cuda")
    cos, sin = tables(5, 64, "cuda")
    for eps in (0.0, 1e-6):
        got, want = (qk_norm_rope(q, q, cos, sin, query_weight=w, key_weight=w, eps=eps,
                                  backend=b)[0] for b in ("triton", "torch"))
        torch.testing.assert_close(got, want, rtol=2 * HALF[dtype] * 2, atol=1e-6, equal_nan=True)


@pytest.mark.gpu
def test_kernel_gradients_of_a_part():
    """Weights without gradients, one input alone, an output that is not used."""
    q, k, gq, gk, wq, wk = inputs(1, 4, 2, 33, 64, torch.float16, 4, device="cuda")
    cos, sin = tables(33, 64, "cuda")
    wq, wk = wq.half().cuda(), wk.half().cuda()
    full = [t.detach().requires_grad_() for t in (q, k, wq, wk)]

    def run(leaves):
        return qk_norm_rope(*leaves[:2], cos, sin, query_weight=leaves[2], key_weight=leaves[3],
                            backend="triton")

    want = torch.autograd.grad(run(full), full, (gq, gk))
    for part in ((0,), (1,), (2,), (3,), (0, 3)):
        leaves = [t.detach().requires_grad_(i in part) for i, t in enumerate(full)]
        got = torch.autograd.grad(run(leaves), [leaves[i] for i in part], (gq, gk))
        for i, g in zip(part, got):
            assert torch.equal(g, want[i]), i
    (dq,) = torch.autograd.grad(run(full)[0], full[0], gq)
    assert torch.equal(dq, want[0])


@pytest.mark.gpu
def test_kernel_calls_repeat_bit_for_bit_on_other_streams_and_in_graphs():
    q, k, gq, gk, wq, wk = inputs(2, 8, 4, 130, 128, torch.bfloat16, 6, device="cuda")
    cos, sin = tables(130, 128, "cuda")
    leaves = [t.detach().requires_grad_() for t in (q, k, wq.bfloat16().cuda(), wk.bfloat16().cuda())]

    def step():
        out = qk_norm_rope(*leaves[:2], cos, sin, query_weight=leaves[2], key_weight=leaves[3],
                           backend="triton")
        return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, (gq, gk)))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(3):
        with torch.no_grad():
            leaves[0].copy_(torch.randn_like(leaves[0]))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want)), i


@pytest.mark.gpu
def test_kernel_reads_tables_as_views_of_complex_numbers():
    """cos and sin as parts of one complex tensor, conjugated: lazily negated and strided."""
    turns = torch.polar(torch.ones(9, 16), torch.randn(9, 16, generator=torch.Generator()
                                                       .manual_seed(3))).cuda().conj()
    q = torch.randn(1, 2, 9, 32, generator=torch.Generator().manual_seed(4)).half().cuda()
    for sin in (turns.imag, torch._neg_view(-turns.imag.clone())):
        assert sin.is_neg()
        got, other = both_paths(lambda: qk_norm_rope(q, q, turns.real, sin, backend="triton")[0])
        want = qk_norm_rope(q, q, turns.real.clone(), sin.resolve_neg().clone(), backend="triton")[0]
        assert torch.equal(got, want) and torch.equal(other, want)


def both_paths(call):
    """call() through the C++ binding and through the Python op layer."""
    assert _native.available(), _native.status()[1]
    got = call()
    with pytest.MonkeyPatch.context() as m:
        m.setattr(_native, "available", lambda: False)
        other = call()
    return got, other


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [True, False])
def test_binding_and_op_layer_agree_bit_for_bit(norm):
    q, k, gq, gk, wq, wk = inputs(2, 8, 4, 70, 96, torch.bfloat16, 8, "tokens", "cuda")
    cos, sin = tables(90, 64, "cuda")
    pos = positions_of("each", 2, 70, 90).cuda()
    leaves = [t.detach().requires_grad_() for t in (q, k)]
    weights = {}
    if norm:
        leaves += [w.cuda().requires_grad_() for w in (wq, wk)]
        weights = dict(query_weight=leaves[2], key_weight=leaves[3])

    def call():
        out = qk_norm_rope(leaves[0], leaves[1], cos, sin, positions=pos, backend="triton", **weights)
        with torch.no_grad():
            plain = qk_norm_rope(leaves[0], leaves[1], cos, sin, positions=pos, **weights)
        return [*out, *plain, *torch.autograd.grad(out, leaves, (gq, gk))]

    for a, b in zip(*both_paths(call)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_kernel_has_no_second_derivative():
    q, k, gq, gk, _, _ = inputs(1, 2, 1, 8, 32, torch.float16, 9, device="cuda")
    cos, sin = tables(8, 32, "cuda")
    q.requires_grad_()

    def call():
        out, _ = qk_norm_rope(q, k, cos, sin, backend="triton")
        (g,) = torch.autograd.grad(out, q, gq.requires_grad_(), create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), gq)
        return g.detach()

    a, b = both_paths(call)
    assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("eps", [1e-6, 0])  # an int goes through the Python Function
def test_capture_beside_a_living_graph_of_the_same_leaves_is_refused(eps):
    q, k, gq, gk, _, _ = inputs(1, 2, 1, 8, 32, torch.float16, 9, device="cuda")
    cos, sin = tables(8, 32, "cuda")
    q.requires_grad_()
    alive, _ = qk_norm_rope(q, k, cos, sin, eps=eps, backend="triton")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = gq + 0  # the graph is not empty
        with pytest.raises(RuntimeError, match="same leaf tensors"):
            qk_norm_rope(q, k, cos, sin, eps=eps, backend="triton")
    want = torch.autograd.grad(alive, q, gq)[0]
    del alive, _
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        out, _ = qk_norm_rope(q, k, cos, sin, eps=eps, backend="triton")
        torch.autograd.grad(out, q, gq)
    del out, _
    out, _ = qk_norm_rope(q, k, cos, sin, eps=eps, backend="triton")
    assert torch.equal(torch.autograd.grad(out, q, gq)[0], want)
    assert z.shape == gq.shape


@pytest.mark.gpu
def test_kernel_refuses_what_it_cannot_serve():
    cos, sin = tables(4, 12, "cuda")
    q = torch.randn(1, 2, 4, 32, device="cuda").half()
    with pytest.raises(RuntimeError, match="multiple of 16"):
        qk_norm_rope(q, q, cos, sin, backend="triton")
    cos, sin = tables(4, 16, "cuda")
    with pytest.raises(RuntimeError, match="float16 and bfloat16"):
        qk_norm_rope(q.float(), q.float(), cos, sin, backend="triton")
    with pytest.raises(RuntimeError, match="multiple of 8"):
        qk_norm_rope(q[..., :20], q[..., :20], cos[:, :8], sin[:, :8], backend="triton")
    with pytest.raises(RuntimeError, match="derivative in cos"):
        qk_norm_rope(q, q, cos.requires_grad_(), sin, backend="triton")


@pytest.mark.gpu
def test_eps_outside_float32():
    """PyTorch serves it (the norm's root is infinite); the kernel says why it does not."""
    q = torch.randn(1, 2, 4, 32, device="cuda").half()
    w = torch.ones(32, device="cuda")
    args = (q, q, *tables(4, 16, "cuda"))
    for eps in (1e39, 10 ** 40):
        weights = dict(query_weight=w, key_weight=w, eps=eps)
        got, want = (qk_norm_rope(*args, backend=b, **weights)[0] for b in ("auto", "torch"))
        assert torch.equal(got, want) and not want.any()
        with pytest.raises(RuntimeError, match="outside float32"):
            qk_norm_rope(*args, backend="triton", **weights)
    weights["eps"] = 3e38
    got, want = (qk_norm_rope(*args, backend=b, **weights)[0] for b in ("triton", "torch"))
    assert torch.equal(got, want)
