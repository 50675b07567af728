"""The operators around the attention call: what a decoder layer does to queries and keys
before it, and the paged key/value cache that a serving program keeps for it.

A case is one call (or one training step) of one of them, named by ``op``:

  rope    ``qk_norm_rope``: RMS norm of each head's queries and keys, and their rotation by
          position, in one pass; ``train`` takes the gradients too
  plan    ``paged_cache_plan``: pages and cache slots of a step's new tokens, from the lengths
  store   ``paged_cache_store``: keys and values of new tokens into their slots
  attend  ``paged_attention``: the attention of the newest tokens over the paged cache

``own`` chooses between the plain form of each (elementary torch operations in 32 bits) and
the package's call; ``exact`` is its definition in 64 bits.

Case fields:
  B, Hq, Hkv, N, D      sequences, query and key/value heads, tokens a sequence, head size
  T                     store: tokens of the step, padding included
  page                  tokens of a page
  lo, hi                range of the sequences' lengths (rope: hi is the length of the tables)
  new_lo, new_hi        plan: range of the sequences' new tokens
  dtype                 "float16" or "bfloat16"
  layout                rope, store: "heads" (contiguous [B, H, N, D]) or "tokens" (views of the
                        projections' [B, N, H, D]); the cache: "heads" ([pages, H, page, D]) or
                        "tokens" (views of [pages, page, H, D])
  norm, rotary, interleaved, train   rope's form
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_PACKAGE = str(Path(__file__).resolve().parent.parent / "triton-flash-attention_amd")


def _api():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    import triton_flash_attention

    return triton_flash_attention


# ---- the cases --------------------------------------------------------------------------


def _rope(B, Hq, Hkv, N, D, dtype, layout, *, norm=True, rotary=None, interleaved=False,
          train=False, hi=None, **name):
    return dict(op="rope", B=B, Hq=Hq, Hkv=Hkv, N=N, D=D, dtype=dtype, layout=layout, norm=norm,
                rotary=rotary or D, interleaved=interleaved, train=train, hi=hi or N, **name)


def _plan(B, lo, hi, new_lo, new_hi, page, **name):
    return dict(op="plan", B=B, lo=lo, hi=hi, new_lo=new_lo, new_hi=new_hi, page=page, **name)


def _store(T, Hkv, D, dtype, layout, page, **name):
    return dict(op="store", T=T, Hkv=Hkv, D=D, dtype=dtype, layout=layout, page=page, **name)


def _attend(B, Hq, Hkv, N, D, dtype, layout, page, lo, hi, **name):
    return dict(op="attend", B=B, Hq=Hq, Hkv=Hkv, N=N, D=D, dtype=dtype, layout=layout, page=page,
                lo=lo, hi=hi, **name)


def listed():
    return [
        # The new token of each of eight sequences, on its way to the cache.
        _rope(8, 32, 8, 1, 128, "bfloat16", "tokens", hi=8192, name="rope_step"),
        # One prompt of odd length, rotated without norms: inference.
        _rope(1, 32, 8, 3001, 128, "float16", "tokens", norm=False, name="rope_prompt"),
        # A decoder layer's training step on the projections' views.
        _rope(2, 32, 8, 2048, 128, "bfloat16", "tokens", train=True, name="rope_train"),
        # Long sequences with small heads of which half is rotated, in neighbouring pairs.
        _rope(4, 16, 16, 4096, 64, "float16", "heads", rotary=32, interleaved=True, train=True,
              name="rope_train_partial"),
        # One new token for each running sequence.
        _plan(64, 1, 8192, 1, 1, 16, name="plan_step"),
        # Prompts of every length join sequences of every length.
        _plan(509, 0, 4096, 0, 2049, 16, name="plan_prompts"),
        # The keys and values of one step, and of a long prompt from a fused projection.
        _store(32, 8, 128, "bfloat16", "heads", 16, name="store_step"),
        _store(16381, 8, 128, "float16", "tokens", 16, name="store_prompt"),
        # The smallest attention call: one short sequence, latency counts.
        _attend(1, 32, 8, 1, 128, "float16", "heads", 16, 257, 257, name="attend_one"),
        # A running batch: sequences from a few tokens to thousands.
        _attend(32, 32, 8, 1, 128, "bfloat16", "heads", 16, 17, 8192, name="attend_ragged"),
        # Four drafted tokens are checked at once, a head of keys for each head of queries.
        _attend(16, 16, 16, 4, 64, "float16", "tokens", 32, 257, 3001, name="attend_draft"),
        # The largest: a batch of long sequences.
        _attend(8, 32, 8, 1, 128, "float16", "heads", 64, 32768, 32768, name="attend_long"),
    ]


# The most values that a drawn rope case holds, and the most of keys, and of pairs of queries
# and keys, times the head size in a drawn attention case: those of the largest listed ones.
_MOST_ROPE = 2 * 40 * 2048 * 128
_MOST_KEYS = 8 * 32768 * 8 * 128
_MOST_PAIRS = 8 * 32768 * 32 * 128


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    while True:
        op = rng.choice(["rope", "rope", "plan", "store", "attend", "attend", "attend"])
        dtype = rng.choice(["float16", "bfloat16"])
        layout = rng.choice(["heads", "tokens"])
        D = rng.choice([32, 64, 64, 128, 128, 128, 80, 96])
        Hkv = rng.choice([1, 2, 4, 8, 16])
        Hq = min(32, Hkv * rng.choice([1, 2, 4, 8]))
        page = rng.choice([16, 16, 32, 48, 64, 128])
        if op == "rope":
            train = rng.random() < 0.5
            N = _log_int(rng, 16, 8192) if train else rng.choice([1, 1, _log_int(rng, 2, 8192)])
            B = _log_int(rng, 1, 64 if N == 1 else 8)
            if B * (Hq + Hkv) * N * D > _MOST_ROPE:
                continue
            return _rope(B, Hq, Hkv, N, D, dtype, layout, norm=rng.random() < 0.7,
                         rotary=rng.choice([D, D, 16 * max(1, D // 32)]),
                         interleaved=rng.random() < 0.3, train=train,
                         hi=max(N, _log_int(rng, 256, 16384)))
        if op == "plan":
            B, new = _log_int(rng, 1, 509), rng.choice([1, 4, _log_int(rng, 1, 2049)])
            return _plan(B, rng.choice([0, 1]), _log_int(rng, 16, 4096),
                         rng.choice([0, new]), new, page)
        if op == "store":
            return _store(_log_int(rng, 1, 16381), min(8, Hkv), D, dtype, layout, page)
        hi = _log_int(rng, 16, 32768)
        lo = rng.choice([1, max(1, hi // 2), hi])
        B, N = _log_int(rng, 1, 64), rng.choice([1, 1, 1, 2, 5])
        if B * hi * Hkv * D <= _MOST_KEYS and B * N * hi * Hq * D <= _MOST_PAIRS:
            return _attend(B, Hq, Hkv, N, D, dtype, layout, page, lo, hi)


# ---- their inputs -----------------------------------------------------------------------


def _spread(n, lo, hi, offset=0.0):
    """n whole numbers spread over [lo, hi] in no order; the first (offset 0) is hi."""
    return [hi - int((hi - lo + 1) * ((0.6180339887498949 * i + offset) % 1.0)) for i in range(n)]


def _lengths(case):
    return _spread(case["B"], case["lo"], case["hi"])


def _new(case):
    return _spread(case["B"], case["new_lo"], case["new_hi"], 0.37)


def _cdiv(a, b):
    return -(-a // b)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _cache(case, pages, gen, dtype):
    """An empty or filled cache [pages, Hkv, page, D] in the case's layout."""
    H, S, D = case["Hkv"], case["page"], case["D"]
    if case["layout"] == "tokens":
        shape = (pages, S, H, D)
    else:
        shape = (pages, H, S, D)
    t = torch.empty(shape, dtype=dtype, device="cuda")
    t.normal_(generator=gen)
    return t.transpose(1, 2) if case["layout"] == "tokens" else t


def _prepare_rope(case, gen, dtype):
    B, N, D, R = case["B"], case["N"], case["D"], case["rotary"]
    shapes = [(B, case[h], N, D) for h in ("Hq", "Hkv")]
    if case["layout"] == "tokens":  # slices of one fused projection
        heads = case["Hq"] + case["Hkv"]
        fused = _randn(gen, (B, N, heads, D), dtype)
        q, k = fused[:, :, :case["Hq"]].transpose(1, 2), fused[:, :, case["Hq"]:].transpose(1, 2)
    else:
        q, k = (_randn(gen, s, dtype) for s in shapes)
    state = {"q": q, "k": k, "wq": None, "wk": None}
    if case["norm"]:
        for w in ("wq", "wk"):
            state[w] = (1 + 0.25 * torch.randn(D, generator=gen, device="cuda")).to(dtype)
    # The tables of every program: angles in 64 bits, kept in 32.
    angle = torch.arange(case["hi"], dtype=torch.float64, device="cuda")[:, None] * torch.pow(
        torch.tensor(10000.0, dtype=torch.float64, device="cuda"),
        -torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)
    state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    # Decoding: each sequence is at a place of its own; otherwise tokens 0 .. N - 1.
    state["positions"] = None
    if N == 1:
        state["positions"] = torch.randint(0, case["hi"], (B, 1), generator=gen, device="cuda")
    if case["train"]:
        state["gq"], state["gk"] = (_randn(gen, s, dtype) for s in shapes)
        for n in ("q", "k", "wq", "wk"):
            if state[n] is not None:
                state[n] = state[n].detach().requires_grad_()
    return state


def _prepare_plan(case, gen, dtype):
    B, S = case["B"], case["page"]
    lengths, new = _lengths(case), _new(case)
    held = [_cdiv(n, S) for n in lengths]
    need = sum(_cdiv(n + k, S) - h for n, k, h in zip(lengths, new, held))
    width = max(max(_cdiv(n + k, S) for n, k in zip(lengths, new)), 1)
    pages = torch.randperm(sum(held) + need + 8, generator=gen, device="cuda").int()
    used, free = pages[:sum(held)], pages[sum(held):]
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    rows = torch.repeat_interleave(torch.arange(B, device="cuda"), _ints(held, torch.int64))
    first = torch.cumsum(_ints(held, torch.int64), 0) - _ints(held, torch.int64)
    table[rows, torch.arange(sum(held), device="cuda") - first[rows]] = used
    return {"table": table, "lengths": _ints(lengths), "new": _ints(new), "free": free.contiguous(),
            "tokens": max(1, _cdiv(sum(new), 64) * 64)}


def _prepare_store(case, gen, dtype):
    T, H, D, S = case["T"], case["Hkv"], case["D"], case["page"]
    pages = _cdiv(T, S) * 2 + 1
    if case["layout"] == "tokens":
        fused = _randn(gen, (T, 6 * H, D), dtype)  # queries (four a head), keys, values
        key, value = fused[:, 4 * H:5 * H], fused[:, 5 * H:]
    else:
        key, value = (_randn(gen, (T, H, D), dtype) for _ in range(2))
    slots = torch.randperm(pages * S, generator=gen, device="cuda")[:T]
    slots[T - T // 8:] = -1  # a padded step
    caches = [_cache(dict(case, layout="heads"), pages, gen, dtype) for _ in range(2)]
    return {"key": key, "value": value, "kc": caches[0], "vc": caches[1], "slots": slots}


def _prepare_attend(case, gen, dtype):
    B, S = case["B"], case["page"]
    lengths = _lengths(case)
    width = _cdiv(max(lengths), S)
    pages = sum(_cdiv(n, S) for n in lengths) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").int().tolist()
    table, at = [], 0
    for n in lengths:
        held = _cdiv(n, S)
        table.append(order[at:at + held] + [-1] * (width - held))
        at += held
    q = _randn(gen, (B, case["Hq"], case["N"], case["D"]), dtype)
    kc, vc = (_cache(case, pages, gen, dtype) for _ in range(2))
    return {"q": q, "kc": kc, "vc": vc, "table": _ints(table), "lengths": _ints(lengths)}


_PREPARE = {"rope": _prepare_rope, "plan": _prepare_plan, "store": _prepare_store,
            "attend": _prepare_attend}


def prepare(case, seed):
    dtype = getattr(torch, case.get("dtype", "float16"))
    state = _PREPARE[case["op"]](case, _gen(seed), dtype)
    state["case"] = case
    return state


# ---- one pass ---------------------------------------------------------------------------


def _rotate(y, cos, sin, interleaved):
    """The first 2 cos.shape[-1] values of y's rows rotated."""
    R = 2 * cos.shape[-1]
    x, rest = y[..., :R], y[..., R:]
    a, b = (x[..., ::2], x[..., 1::2]) if interleaved else (x[..., :R // 2], x[..., R // 2:])
    z = (a * cos - b * sin, b * cos + a * sin)
    z = torch.stack(z, -1).flatten(-2) if interleaved else torch.cat(z, -1)
    return torch.cat((z, rest), -1)


def _plain_rope(x, w, cos, sin, interleaved, eps):
    y = x.float()
    if w is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * w.float()
    return _rotate(y, cos, sin, interleaved).to(x.dtype).contiguous()


def _run_rope(s, c):
    if own:
        q, k = _api().qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], query_weight=s["wq"],
                                   key_weight=s["wk"], eps=1e-6, positions=s["positions"],
                                   interleaved=c["interleaved"], backend="triton")
    else:
        if s["positions"] is None:
            cos, sin = s["cos"][:c["N"]], s["sin"][:c["N"]]
        else:
            cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]
        q, k = (_plain_rope(x, w, cos, sin, c["interleaved"], 1e-6)
                for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])))
    if not c["train"]:
        return {"q": q, "k": k}
    names = [n for n in ("q", "k", "wq", "wk") if s[n] is not None]
    grads = torch.autograd.grad((q, k), [s[n] for n in names], (s["gq"], s["gk"]))
    return {"q": q.detach(), "k": k.detach(), **{"d" + n: g for n, g in zip(names, grads)}}


def _run_plan(s, c):
    if own:
        p = _api().paged_cache_plan(s["table"], s["lengths"], s["new"], s["free"],
                                    page_size=c["page"], num_tokens=s["tokens"], backend="triton")
        return {"table": s["table"], "slots": p.slots, "positions": p.positions,
                "starts": p.starts, "lengths": p.lengths, "free_start": p.free_start}
    S, table, lengths, new = c["page"], s["table"], s["lengths"].long(), s["new"].long()
    held = (lengths + S - 1) // S
    need = (lengths + new + S - 1) // S - held
    ends, taken = torch.cumsum(new, 0), torch.cumsum(need, 0)
    starts = torch.cat((torch.zeros_like(ends[:1]), ends))
    # every place that a new page could take: its place in the list of free pages
    j = torch.arange(table.shape[1], device=table.device) - held[:, None]
    at = torch.where((j >= 0) & (j < need[:, None]), (taken - need)[:, None] + j, -1)
    table.copy_(torch.where(at >= 0, s["free"][at.clamp(0, s["free"].shape[0] - 1)], table))
    t = torch.arange(s["tokens"], device=table.device)
    row = (t[:, None] >= ends[None, :]).sum(1).clamp(max=c["B"] - 1)
    valid = t < ends[-1]
    position = torch.where(valid, lengths[row] + t - starts[row], 0)
    slots = table[row, position // S].long() * S + position % S
    return {"table": table, "slots": torch.where(valid, slots, -1), "positions": position.int(),
            "starts": starts.int(), "lengths": (lengths + new).int(), "free_start": taken[-1:].int()}


def _run_store(s, c):
    if own:
        _api().paged_cache_store(s["key"], s["value"], s["kc"], s["vc"], s["slots"],
                                 backend="triton")
    else:
        # padding rows write what the first row writes
        rows = torch.where(s["slots"] >= 0, torch.arange(c["T"], device="cuda"), 0)
        page, at = s["slots"][rows] // c["page"], s["slots"][rows] % c["page"]
        s["kc"][page, :, at] = s["key"][rows]
        s["vc"][page, :, at] = s["value"][rows]
    return {"k": s["kc"], "v": s["vc"]}


def _run_attend(s, c):
    if own:
        return {"o": _api().paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["lengths"],
                                            enable_gqa=c["Hq"] != c["Hkv"], backend="triton")}
    B, Hq, N, D = s["q"].shape
    H, S, M = c["Hkv"], c["page"], s["table"].shape[1]
    q = s["q"].float().reshape(B, H, Hq // H * N, D)  # the rows that read one key head
    last = (s["lengths"][:, None] - N + torch.arange(N, device=q.device)).repeat(1, Hq // H)
    keys = torch.arange(M * S, device=q.device)
    out = []
    for b in range(B):
        pages = s["table"][b].clamp(min=0)
        k, v = (t[pages].transpose(0, 1).reshape(H, M * S, D).float() for t in (s["kc"], s["vc"]))
        seen = keys <= last[b][:, None]
        scores = torch.matmul(q[b], k.transpose(1, 2).contiguous()) * D ** -0.5
        scores = scores.masked_fill(~seen, -math.inf)
        m = scores.amax(-1, keepdim=True)
        p = torch.exp(scores - torch.where(m == -math.inf, 0.0, m))
        total = p.sum(-1, keepdim=True)
        out.append(torch.matmul(p / torch.where(total > 0, total, 1.0), v))
    return {"o": torch.stack(out).reshape(B, Hq, N, D).to(s["q"].dtype)}


_RUN = {"rope": _run_rope, "plan": _run_plan, "store": _run_store, "attend": _run_attend}


def run(state):
    return _RUN[state["case"]["op"]](state, state["case"])


# ---- what a pass cannot do without ------------------------------------------------------


def work(case):
    op = case["op"]
    if op == "rope":
        values = case["B"] * (case["Hq"] + case["Hkv"]) * case["N"] * case["D"]
        tables = min(case["hi"], case["B"] if case["N"] == 1 else case["N"]) * case["rotary"] * 4
        # read and written once; training reads q, k, their outputs' gradients (and q and k
        # once more where a norm's gradient needs them) and writes both gradients
        passes = 2 if not case["train"] else (5 if case["norm"] else 4)
        return {"bytes": 2 * passes * values + tables, "flops": 6 * passes * values}
    if op == "plan":
        tokens, S = sum(_new(case)), case["page"]
        pages = sum(_cdiv(n + k, S) - n // S for n, k in zip(_lengths(case), _new(case)) if k)
        # a slot and a position a token, a page id read and written a page, the lengths
        return {"bytes": 12 * tokens + 8 * pages + 20 * case["B"], "flops": 8 * tokens}
    if op == "store":
        return {"bytes": (case["T"] - case["T"] // 8) * 8 * case["Hkv"] * case["D"] + 8 * case["T"],
                "flops": 0}
    q = case["B"] * case["Hq"] * case["N"] * case["D"]
    keys = sum(_lengths(case))
    return {"bytes": 4 * q + 4 * keys * case["Hkv"] * case["D"] + 4 * keys // case["page"],
            "flops": 4 * keys * case["Hq"] * case["N"] * case["D"]}


# ---- the definitions in 64 bits ---------------------------------------------------------


def _exact_rope(s, c):
    B, N, D, R = c["B"], c["N"], c["D"], c["rotary"]
    place = torch.arange(N, device="cuda").expand(B, N) if s["positions"] is None else s["positions"]
    # the rotation as a product of complex numbers
    turn = torch.complex(s["cos"].double(), s["sin"].double())[place][:, None]

    def split(t):
        t = t[..., :R]
        if c["interleaved"]:
            return torch.view_as_complex(t.reshape(*t.shape[:-1], R // 2, 2).contiguous())
        return torch.complex(t[..., :R // 2].contiguous(), t[..., R // 2:].contiguous())

    def join(z, t):
        r = torch.view_as_real(z)
        r = r.flatten(-2) if c["interleaved"] else torch.cat((r[..., 0], r[..., 1]), -1)
        return torch.cat((r, t[..., R:]), -1)

    out = {}
    for n in ("q", "k"):
        x = s[n].detach().double()
        w = None if s["w" + n] is None else s["w" + n].detach().double()
        unit = x
        if w is not None:
            inv = 1.0 / torch.sqrt((x * x).sum(-1, keepdim=True) / D + 1e-6)
            unit = x * inv
        y = unit if w is None else unit * w
        out[n] = join(split(y) * turn, y)
        if not c["train"]:
            continue
        g = s["g" + n].double()
        u = join(split(g) * turn.conj(), g)
        if w is None:
            out["d" + n] = u
        else:
            out["dw" + n] = (u * unit).sum((0, 1, 2))
            t = u * w
            out["d" + n] = inv * (t - unit * (t * unit).mean(-1, keepdim=True))
    order = ["q", "k"] + [n for n in ("dq", "dk", "dwq", "dwk") if n in out]
    return {n: out[n] for n in order}


def _exact_plan(s, c):
    S, table = c["page"], s["table"].cpu()
    free, lengths, new = s["free"].tolist(), s["lengths"].tolist(), s["new"].tolist()
    slots, positions, starts, at = [], [], [0], 0
    for b, (n, k) in enumerate(zip(lengths, new)):
        for j in range(_cdiv(n, S), _cdiv(n + k, S)):
            table[b, j] = free[at]
            at += 1
        row = table[b].tolist()
        slots += [row[p // S] * S + p % S for p in range(n, n + k)]
        positions += range(n, n + k)
        starts.append(len(slots))
    pad = s["tokens"] - len(slots)
    return {"table": table.cuda(), "slots": _ints(slots + [-1] * pad, torch.int64),
            "positions": _ints(positions + [0] * pad), "starts": _ints(starts),
            "lengths": _ints([n + k for n, k in zip(lengths, new)]), "free_start": _ints([at])}


def _exact_store(s, c):
    out, slots = {}, s["slots"]
    for n, t, cache in (("k", s["key"], s["kc"]), ("v", s["value"], s["vc"])):
        flat = cache.transpose(1, 2).reshape(-1, c["Hkv"], c["D"]).clone()
        kept = slots >= 0
        flat.index_copy_(0, slots[kept], t[kept])
        out[n] = flat.view(-1, c["page"], c["Hkv"], c["D"]).transpose(1, 2).double()
    return out


def _exact_attend(s, c):
    B, Hq, N, D = s["q"].shape
    H, S = c["Hkv"], c["page"]
    out = torch.zeros(B, Hq, N, D, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(c)):
        at = torch.arange(n, device="cuda")
        page, row = s["table"][b].long()[at // S], at % S
        for h in range(H):
            k, v = (t[page, h, row].double() for t in (s["kc"], s["vc"]))
            heads = slice(h * (Hq // H), (h + 1) * (Hq // H))
            for i in range(N):
                seen = n - N + i + 1
                if seen > 0:
                    p = torch.softmax(s["q"][b, heads, i].double() @ k[:seen].t() / math.sqrt(D), -1)
                    out[b, heads, i] = p @ v[:seen]
    return {"o": out}


_EXACT = {"rope": _exact_rope, "plan": _exact_plan, "store": _exact_store, "attend": _exact_attend}


def exact(case, seed):
    # The small steps of the 64-bit form take about a millisecond: many of them are left out.
    if case["op"] == "attend" and case["B"] * case["Hkv"] * case["N"] > 8000:
        return None
    return _EXACT[case["op"]](prepare(case, seed), case)
