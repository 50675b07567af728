"""Attention over shared prefixes where its work spreads over the whole chip: rows of thousands of
pieces, prefixes that are cut into pieces, and the memory that a call may write. Where the pieces lie is
read from the calls' workspaces, so that no case leaves its path unseen, and compared with the walk of
test_prefix_line.py."""

from __future__ import annotations

import pytest
import torch
from test_paged import F32, HALF
from test_prefix import make_shared, within
from test_prefix_line import Line

from triton_flash_attention import _lib, _native, _ops, paged_prefix_attention


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


GUARD = 4096


class Workspaces:
    """Calls of the op layer whose workspaces lie between guards, exactly as long as the calls ask."""

    def __init__(self, monkeypatch):
        self.kept = []
        launch = _ops._launch

        def guarded(name, entry, *args):
            n = args[-2]
            room = torch.full((n + 2 * GUARD,), 0xA5, dtype=torch.uint8, device="cuda")
            self.kept.append((room, n))
            return launch(name, entry, *args[:-3], room.data_ptr() + GUARD, n, args[-1])

        monkeypatch.setattr(_native, "available", lambda: False)
        monkeypatch.setattr(_native, "module", lambda: None)
        monkeypatch.setattr(_ops, "_launch", guarded)

    def last(self):
        """The last call's workspace, as int32, with its guards as they were."""
        room, n = self.kept.pop()
        assert bool((room[:GUARD] == 0xA5).all()) and bool((room[GUARD + n:] == 0xA5).all())
        return room[GUARD:GUARD + n // 4 * 4].view(torch.int32).cpu()


def reference_on_gpu(q, dense, scale, dtype):
    """attention_reference of test_paged.py with its products on the GPU, in 64 bits as well."""
    B, Hq, N, D = q.shape
    o, bound = (torch.zeros(B, Hq, N, D, dtype=torch.float64) for _ in range(2))
    for b, (k, v) in enumerate(dense):
        n, H = k.shape[:2]
        if n == 0:
            continue
        k, v = (t.to("cuda").transpose(0, 1).contiguous() for t in (k, v))  # [H, n, D]
        x = q[b].to("cuda").double().reshape(H, Hq // H * N, D)
        last = n - N + torch.arange(N, device="cuda").repeat(Hq // H)
        seen = torch.arange(n, device="cuda")[None] <= last[:, None]
        s = torch.matmul(x, k.transpose(1, 2).contiguous()) * scale
        size = torch.matmul(x.abs(), k.abs().transpose(1, 2).contiguous()) * abs(scale)
        d = (136 * size.masked_fill(~seen, 0).amax(-1) + 8 * s.masked_fill(~seen, 0).abs().amax(-1)) * F32
        m = s.masked_fill(~seen, -1e300).amax(-1, keepdim=True)
        p = torch.where(seen, torch.exp(s - m), 0.0)
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total == 0, 1.0, total)
        A = torch.matmul(p, v.abs())
        small = 2.0 ** -32 * torch.matmul(seen.double()[None].expand(H, -1, -1).contiguous(), v.abs())
        o[b] = torch.matmul(p, v).reshape(Hq, N, D).cpu()
        counted = (last + 1).clamp(min=0)[None, :, None]
        e = A * (HALF[dtype] + counted * F32 + 4 * d[..., None])
        bound[b] = (e + (small if dtype == torch.float16 else 0)).reshape(Hq, N, D).cpu()
    return o, bound


def places(ws, line):
    """The places that a call left in its workspace, and those that the walk has for it."""
    B, G = line.B, line.G
    seqs = ws[16:16 + 4 * B].reshape(B, 4).tolist()
    groups = ws[16 + 4 * B:16 + 4 * B + 8 * G].reshape(G, 8)[:, :5].tolist()
    return (ws[:4].tolist(), [tuple(t) for t in seqs], [tuple(t) for t in groups]), (
        [line.L, line.own_stretch, 0, line.pieces], line.seqs, line.groups)


F16, BF16 = torch.float16, torch.bfloat16
_own = [3000 + 137 * i for i in range(48)]
PIECES = [
    # what it is for; sizes, prefixes, lengths, Hq, Hkv, N, D, S, type
    ("one tile, a prefix that ends inside a page",
     [3], [36805], [36810, 36900, 36806], 16, 8, 1, 32, 64, F16),
    ("one tile, two key groups", [2], [50000], [50010, 50100], 8, 4, 1, 128, 32, BF16),
    ("tiles, few rows a sequence",
     [40], [13001], [13001 + i for i in range(40)], 8, 2, 9, 64, 16, BF16),
    ("tiles, many rows a sequence",
     [12], [25001], [25001 + 40 * i for i in range(12)], 2, 1, 40, 128, 48, F16),
    ("long and short prefixes", [2, 30, 1, 3], [30000, 9000, 100, 50],
     [30900, 31000] + [9000 + 30 * i for i in range(30)] + [77, 50, 90, 3000], 8, 2, 10, 64, 64, F16),
    ("long and short prefixes, many rows a sequence", [2, 3, 4, 2], [24000, 9000, 60, 13000],
     [24500, 24001, 9000, 9700, 9001, 60, 100, 61, 300, 13000, 13001, 2000, 2000, 1], 16, 2, 9, 128, 16,
     BF16),
    ("heavy own keys, and members shorter than the prefix", [6, 2], [9000, 500],
     [9001, 12999, 4000, 9000, 0, 8999, 800, 501] + _own, 4, 4, 2, 128, 32, F16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", PIECES, ids=[c[0] for c in PIECES])
def test_long_prefixes_in_pieces(case, monkeypatch):
    sizes, prefix, lengths, Hq, Hkv, N, D, S, dtype = case[1:]
    views, table, starts, dense = make_shared(sizes, prefix, lengths, Hkv, S, D, dtype, device="cuda")
    q = torch.randn(len(lengths), Hq, N, D, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    kept = Workspaces(monkeypatch)
    o = paged_prefix_attention(q, *views, table, ints(lengths), starts, ints(prefix), enable_gqa=True,
                               backend="triton")
    line = Line(sizes, prefix, lengths, Hkv, Hq // Hkv * N, D, table.shape[1] * S)
    got, want = places(kept.last(), line)
    assert got[0][3] > 0, "no prefix was cut"
    assert got == want
    within(o, *reference_on_gpu(q, dense, D ** -0.5, dtype), dtype)
    monkeypatch.undo()
    again = paged_prefix_attention(q, *views, table, ints(lengths), starts, ints(prefix),
                                   enable_gqa=True, backend="triton")
    assert torch.equal(o, again)


@pytest.mark.gpu
@pytest.mark.parametrize("R", [64, 100])
def test_pieces_that_find_no_room_stay_on_the_line(R, monkeypatch):
    """Own keys that leave the long prefix fewer work-groups than its pieces, which come in eights."""
    if R == 64:
        sizes, prefix, own = [2], [640], [94 * 32] * 53 + [6 * 32]
    else:
        sizes, prefix, own = [3, 3, 3], [384] * 3, [94 * 32] * 59 + [47 * 32]
    lengths, D, S = [prefix[0]] * sum(sizes) + own, 128, 32
    views, table, starts, dense = make_shared(sizes, prefix, lengths, 1, S, D, BF16, device="cuda")
    q = torch.randn(len(lengths), 4, R // 4, D, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    kept = Workspaces(monkeypatch)
    o = paged_prefix_attention(q, *views, table, ints(lengths), starts, ints(prefix), enable_gqa=True,
                               backend="triton")
    line = Line(sizes, prefix, lengths, 1, R, D, table.shape[1] * S)
    assert line.given_up and line.waves == (R == 64)
    got, want = places(kept.last(), line)
    assert got == want
    within(o, *reference_on_gpu(q, dense, D ** -0.5, BF16), BF16)


@pytest.mark.gpu
def test_a_missing_page_inside_a_piece():
    """Pieces begin at any multiple of 32 keys, so inside pages of 64. A page that does not exist makes
    the sequences NaN that need it, and no others."""
    sizes, prefix, lengths, S, D = [3], [36800], [36810, 36900, 10000], 64, 32
    views, table, starts, dense = make_shared(sizes, prefix, lengths, 8, S, D, F16, device="cuda", fill=0.0)
    line = Line(sizes, prefix, lengths, 8, 2, D, table.shape[1] * S)
    begins = {32 * u0 for kind, _, _, u0, _, _ in line.walk() if kind == "prefix"}
    key = min(k for k in begins if k > 10000 + S and k % S == 32)
    q = torch.randn(3, 16, 1, D, generator=torch.Generator().manual_seed(1)).half().cuda()
    want, bound = reference_on_gpu(q, dense, D ** -0.5, F16)
    for bad in (-1, views[0].shape[0], 1 << 30):
        t = table.clone()
        t[0, key // S] = bad
        o = paged_prefix_attention(q, *views, t, ints(lengths), starts, ints(prefix), enable_gqa=True,
                                   backend="triton")
        assert o[:2].isnan().all()
        within(o[2:], want[2:], bound[2:], F16)
    # the page behind the prefix, which ends with a page: the first sequence alone
    t = table.clone()
    t[0, 36800 // S] = -1
    o = paged_prefix_attention(q, *views, t, ints(lengths), starts, ints(prefix), enable_gqa=True,
                               backend="triton")
    assert o[0].isnan().all()
    within(o[1:], want[1:], bound[1:], F16)


@pytest.mark.gpu
@pytest.mark.parametrize("case", [
    ([3, 2], [40, 33], [60, 41, 55, 33, 90], 4, 2, 1, 64, 16, F16),     # 16 work-groups
    ([2] * 40, [200] * 40, [210 + i for i in range(80)], 8, 2, 3, 128, 16, BF16),
    ([], [], [700, 20, 5, 0], 2, 1, 70, 32, 48, F16),                    # no prefixes
])
def test_short_prefixes_stay_inside_their_workspaces(case, monkeypatch):
    sizes, prefix, lengths, Hq, Hkv, N, D, S, dtype = case
    views, table, starts, dense = make_shared(sizes, prefix, lengths, Hkv, S, D, dtype, device="cuda")
    q = torch.randn(len(lengths), Hq, N, D, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    kept = Workspaces(monkeypatch)
    o = paged_prefix_attention(q, *views, table, ints(lengths), starts, ints(prefix), enable_gqa=True,
                               backend="triton")
    got, want = places(kept.last(), Line(sizes, prefix, lengths, Hkv, Hq // Hkv * N, D, table.shape[1] * S))
    assert got == want and got[0][3] == 0
    within(o, *reference_on_gpu(q, dense, D ** -0.5, dtype), dtype)


def test_too_many_groups_are_refused():
    """A work-group looks through all groups, the empty ones too."""
    size = _lib.load().fa_paged_prefix_fwd_workspace_bytes
    assert size(2, (1 << 24) - 1, 4, 2, 1, 64, 100, 16) > 0
    assert size(2, 1 << 24, 4, 2, 1, 64, 100, 16) == _lib.FA_ERR_TOO_LARGE
    assert "too many" in _lib.last_error()


@pytest.mark.gpu
def test_too_many_groups_run_in_pytorch():
    views, table, _, dense = make_shared([2], [20], [40, 33], 2, 16, 32, F16, device="cuda", fill=0.0)
    q = torch.randn(2, 4, 1, 32, generator=torch.Generator().manual_seed(1)).half().cuda()
    starts = torch.zeros((1 << 24) + 1, dtype=torch.int32, device="cuda")
    starts[-1] = 2
    prefix = torch.full((1 << 24,), 20, dtype=torch.int32, device="cuda")
    args = (q, *views, table, ints([40, 33]), starts, prefix)
    with pytest.raises(RuntimeError, match="too many"):
        paged_prefix_attention(*args, enable_gqa=True, backend="triton")
    within(paged_prefix_attention(*args, enable_gqa=True),
           *reference_on_gpu(q, dense, 32 ** -0.5, F16), F16)
