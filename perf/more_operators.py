"""The operators of sequences that share pages of the paged key/value cache: the attention of a
batch over a prefix that its sequences have in common, and what a serving program does to the
pages themselves when it forks, reorders, ends and moves sequences.

A case is one call of one of them, named by ``op``:

  prefix   ``paged_prefix_attention``: the attention of the newest tokens over the cache, where
           each group of sequences shares a prefix that is computed once for all of them
  fork     ``paged_cache_fork``: every row of the page table becomes another row's (beams that are
           reordered, samples of one prompt) or is given up; shared pages are counted, pages that
           nobody holds any more return to the free ones
  copy     ``paged_cache_copy``: keys and values of pages into other pages of the cache
  compact  ``paged_cache_compact``: the pages that are held move to the front of the cache

``own`` chooses between the plain form of each (elementary torch operations in 32 bits) and
the package's call; ``exact`` is its definition in 64 bits.

Case fields:
  G, n_lo, n_hi         groups, and the range of their numbers of sequences
  pre_lo, pre_hi        range of the groups' prefix lengths
  lo, hi                range of the tokens of each sequence behind the prefix
  Hq, Hkv, N, D         query and key/value heads, newest tokens a sequence, head size
  page                  tokens of a page
  dtype                 "float16" or "bfloat16"
  layout                the cache: "heads" ([pages, H, page, D]) or "tokens" (views of
                        [pages, page, H, D])
  end                   fork: the share of the groups that end
  pages, moved          copy: pages of the cache, and pairs of pages that are copied
  part                  copy: whether only the first tokens of each page are copied
  held                  compact: the share of the cache's pages that is held
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


def _prefix(G, n_lo, n_hi, pre_lo, pre_hi, lo, hi, Hq, Hkv, N, D, dtype, layout, page, **name):
    return dict(op="prefix", G=G, n_lo=n_lo, n_hi=n_hi, pre_lo=pre_lo, pre_hi=pre_hi, lo=lo, hi=hi,
                Hq=Hq, Hkv=Hkv, N=N, D=D, dtype=dtype, layout=layout, page=page, **name)


def _fork(G, n_lo, n_hi, pre_lo, pre_hi, lo, hi, page, end, **name):
    return dict(op="fork", G=G, n_lo=n_lo, n_hi=n_hi, pre_lo=pre_lo, pre_hi=pre_hi, lo=lo, hi=hi,
                page=page, end=end, **name)


def _copy(pages, moved, Hkv, D, dtype, layout, page, part, **name):
    return dict(op="copy", pages=pages, moved=moved, Hkv=Hkv, D=D, dtype=dtype, layout=layout,
                page=page, part=part, **name)


def _compact(G, n_lo, n_hi, pre_lo, pre_hi, lo, hi, page, held, **name):
    return dict(op="compact", G=G, n_lo=n_lo, n_hi=n_hi, pre_lo=pre_lo, pre_hi=pre_hi, lo=lo, hi=hi,
                page=page, held=held, **name)


def listed():
    return [
        # The smallest: the four beams of one request over its prompt, latency counts.
        _prefix(1, 4, 4, 512, 512, 5, 60, 32, 8, 1, 128, "float16", "heads", 16,
                name="prefix_beams"),
        # A running batch whose requests all begin with the same instructions.
        _prefix(1, 64, 64, 4096, 4096, 1, 1024, 32, 8, 1, 128, "bfloat16", "heads", 16,
                name="prefix_batch"),
        # Requests of two to seven samples each, prompts of every length, a head of keys a head.
        _prefix(24, 2, 7, 301, 3001, 3, 700, 16, 16, 1, 64, "float16", "tokens", 32,
                name="prefix_samples"),
        # Drafted tokens of many sequences are checked at once.
        _prefix(1, 24, 24, 8192, 8192, 6, 900, 32, 4, 5, 128, "bfloat16", "tokens", 64,
                name="prefix_draft"),
        # The largest: a full batch of questions about one long document.
        _prefix(1, 128, 128, 32768, 32768, 129, 1024, 32, 8, 1, 128, "float16", "heads", 64,
                name="prefix_document"),
        # A step of beam search: the survivors' rows in place of the others'.
        _fork(16, 4, 4, 17, 1025, 3, 90, 16, 0.0, name="fork_beams"),
        # Long sequences in small pages; some requests end, others sample anew.
        _fork(96, 1, 8, 100, 8001, 1, 600, 16, 0.2, name="fork_long"),
        # The begun pages that one step's forks copy, in one layer.
        _copy(4096, 48, 8, 128, "bfloat16", "heads", 16, True, name="copy_step"),
        # Head sizes between the powers of two, heads inside the tokens.
        _copy(1500, 701, 4, 80, "float16", "tokens", 48, True, name="copy_tokens"),
        # A cache is compacted: whole pages move.
        _copy(8192, 2048, 8, 128, "bfloat16", "heads", 64, False, name="copy_compact"),
        # A small cache that has been used for a while, and a whole GPU's.
        _compact(8, 1, 5, 17, 500, 1, 200, 16, 0.6, name="compact_small"),
        _compact(200, 1, 5, 100, 16001, 1, 900, 16, 0.5, name="compact_large"),
    ]


# What a drawn case holds at most: values of keys (or of pairs of queries and keys) times the head
# size of the largest attention, entries of the largest page table, values of the largest copy.
_MOST_KEYS = (32768 + 128 * 600) * 8 * 128
_MOST_PAIRS = 128 * 33400 * 32 * 128
_MOST_PADDED = 128 * 1024 * 8 * 128
_MOST_ENTRIES = 430 * 538
_MOST_COPY = 2048 * 64 * 8 * 128


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    while True:
        op = rng.choice(["prefix", "prefix", "prefix", "fork", "copy", "compact"])
        dtype = rng.choice(["float16", "bfloat16"])
        layout = rng.choice(["heads", "tokens"])
        page = rng.choice([16, 16, 32, 48, 64, 128])
        D = rng.choice([32, 64, 64, 128, 128, 128, 80, 96])
        Hkv = rng.choice([1, 2, 4, 8, 16])
        Hq = min(32, Hkv * rng.choice([1, 2, 4, 8]))
        if op == "copy":
            moved = _log_int(rng, 1, 4096)
            pages = 2 * moved + _log_int(rng, 1, 4096)
            if moved * page * Hkv * D <= _MOST_COPY:
                return _copy(pages, moved, Hkv, D, dtype, layout, page, rng.random() < 0.5)
            continue
        G = rng.choice([1, 1, _log_int(rng, 1, 96)])
        n_hi = _log_int(rng, 1, 128 if G == 1 else 12)
        n_lo = rng.choice([1, n_hi, max(1, n_hi // 2)])
        pre_hi = _log_int(rng, 1, 32768 if op == "prefix" else 8001)
        pre_lo = rng.choice([1, pre_hi, max(1, pre_hi // 2)])
        hi = _log_int(rng, 5, 1024)
        lo = rng.choice([1, max(1, hi // 2)])
        if op == "prefix":
            N = rng.choice([1, 1, 1, 2, 5])
            lo = max(lo, N)
            hi = max(lo, hi)
            B = G * n_hi
            if ((G * pre_hi + B * hi) * Hkv * D <= _MOST_KEYS
                    and B * N * (pre_hi + hi) * Hq * D <= _MOST_PAIRS
                    and B * hi * Hkv * D <= _MOST_PADDED):
                return _prefix(G, n_lo, n_hi, pre_lo, pre_hi, lo, hi, Hq, Hkv, N, D, dtype, layout,
                               page)
        elif G * n_hi * -(-(pre_hi + hi) // page) <= _MOST_ENTRIES:
            sizes = (G, n_lo, n_hi, pre_lo, pre_hi, lo, hi, page)
            if op == "fork":
                return _fork(*sizes, rng.choice([0.0, 0.25]))
            return _compact(*sizes, rng.choice([0.3, 0.6, 0.9]))


# ---- their inputs -----------------------------------------------------------------------


def _spread(n, lo, hi, offset=0.0):
    """n whole numbers spread over [lo, hi] in no order; the first (offset 0) is hi."""
    return [hi - int((hi - lo + 1) * ((0.6180339887498949 * i + offset) % 1.0)) for i in range(n)]


def _sizes(case):
    """Sequences of each group, prefix lengths, and each sequence's length with its prefix."""
    n = _spread(case["G"], case["n_lo"], case["n_hi"])
    pre = _spread(case["G"], case["pre_lo"], case["pre_hi"], 0.21)
    more = _spread(sum(n), case["lo"], case["hi"], 0.43)
    first = [p for p, k in zip(pre, n) for _ in range(k)]
    return n, pre, [p + m for p, m in zip(first, more)]


def _cdiv(a, b):
    return -(-a // b)


def _used_pages(case):
    """Pages that the sequences hold: whole ones of a prefix once for its group."""
    n, pre, lengths = _sizes(case)
    S = case["page"]
    return sum(_cdiv(x, S) for x in lengths) - sum(p // S * (k - 1) for p, k in zip(pre, n))


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _cache(case, pages, gen, dtype):
    """A filled cache [pages, Hkv, page, D] in the case's layout."""
    H, S, D = case["Hkv"], case["page"], case["D"]
    tokens = case["layout"] == "tokens"
    t = torch.empty((pages, S, H, D) if tokens else (pages, H, S, D), dtype=dtype, device="cuda")
    t.normal_(generator=gen)
    return t.transpose(1, 2) if tokens else t


def _paged(case, gen, spare):
    """A page table whose groups share the whole pages of their prefixes, as forks leave it.
    Returns the table, the lengths, the groups' first rows, how many hold each page beyond the
    first, and the pages that are free."""
    S = case["page"]
    n, pre, lengths = _sizes(case)
    rows = _ints(range(sum(n)), torch.int64)
    group = torch.repeat_interleave(_ints(range(case["G"]), torch.int64), _ints(n, torch.int64))
    starts = torch.cumsum(_ints([0] + n, torch.int64), 0)
    held = (_ints(lengths, torch.int64) + S - 1) // S
    shared = (_ints(pre, torch.int64) // S)[group]
    j = torch.arange(_cdiv(max(lengths), S), device="cuda")
    leader = torch.where(j < shared[:, None], starts[:-1][group][:, None], rows[:, None])
    mine = (leader == rows[:, None]) & (j < held[:, None])  # entries that hold a page of their own
    number = torch.cumsum(mine.flatten().long(), 0).reshape(mine.shape) - 1
    used = _used_pages(case)
    pages = used + spare(used, sum(n))
    order = torch.randperm(pages, generator=gen, device="cuda").int()
    table = torch.full(mine.shape, -1, dtype=torch.int32, device="cuda")
    page = order[number[leader, j].clamp(min=0)]
    table = torch.where(j < held[:, None], page, table).contiguous()
    shares = torch.zeros(pages, dtype=torch.int32, device="cuda")
    shares.index_add_(0, table.clamp(min=0).flatten(), (table >= 0).int().flatten())
    shares = (shares - 1).clamp(min=0)
    return table, _ints(lengths), starts.int(), shares, order[used:].contiguous()


def _prepare_prefix(case, gen, dtype):
    table, lengths, starts, shares, _ = _paged(case, gen, lambda used, B: 3)
    q = _randn(gen, (lengths.shape[0], case["Hq"], case["N"], case["D"]), dtype)
    kc, vc = (_cache(case, shares.shape[0], gen, dtype) for _ in range(2))
    return {"q": q, "kc": kc, "vc": vc, "table": table, "lengths": lengths, "starts": starts,
            "prefix": _ints(_sizes(case)[1])}


def _prepare_fork(case, gen, dtype):
    table, lengths, starts, shares, free = _paged(case, gen, lambda used, B: B + 8)
    # Each row's successor descends from a row of its group; the groups that end give theirs up.
    n = starts[1:] - starts[:-1]
    group = torch.repeat_interleave(torch.arange(case["G"], device="cuda"), n.long())
    pick = torch.rand(lengths.shape[0], generator=gen, device="cuda")
    parents = starts[group] + (pick * n[group]).int()
    ends = torch.rand(case["G"], generator=gen, device="cuda") < case["end"]
    parents = torch.where(ends[group], -1, parents).int()
    # Every page has a place in the list: those that are held were taken from its front.
    pages = torch.cat((torch.full((shares.shape[0] - free.shape[0],), -1, dtype=torch.int32,
                                  device="cuda"), free))
    return {"table": table, "lengths": lengths, "parents": parents, "shares": shares, "free": pages,
            "start": _ints([pages.shape[0] - free.shape[0]])}


def _prepare_copy(case, gen, dtype):
    kc, vc = (_cache(case, case["pages"], gen, dtype) for _ in range(2))
    order = torch.randperm(case["pages"], generator=gen, device="cuda").int()
    n = case["moved"]
    tokens = None
    if case["part"]:
        tokens = torch.randint(1, case["page"], (n,), generator=gen, device="cuda").int()
    # a step's rows that need no copy name no pages
    idle = torch.arange(n, device="cuda") % 8 == 7
    sources, targets = (torch.where(idle, -1, t).int() for t in (order[:n], order[n:2 * n]))
    return {"kc": kc, "vc": vc, "sources": sources, "targets": targets, "tokens": tokens}


def _prepare_compact(case, gen, dtype):
    table, _, _, shares, free = _paged(
        case, gen, lambda used, B: max(1, int(used * (1 / case["held"] - 1))))
    return {"table": table, "shares": shares, "free": free}


_PREPARE = {"prefix": _prepare_prefix, "fork": _prepare_fork, "copy": _prepare_copy,
            "compact": _prepare_compact}


def prepare(case, seed):
    dtype = getattr(torch, case.get("dtype", "float16"))
    state = _PREPARE[case["op"]](case, _gen(seed), dtype)
    state["case"] = case
    return state


# ---- one pass ---------------------------------------------------------------------------


def _rows_of(cache, table, first, width):
    """The tokens first[i] .. first[i] + width of the sequence whose pages table[i] names, in 32
    bits: [rows, heads, width, D]."""
    S = cache.shape[2]
    at = first[:, None] + torch.arange(width, device=cache.device)
    column = (at // S).clamp(max=table.shape[1] - 1)
    page = torch.gather(table, 1, column).clamp(min=0)
    return cache[page, :, at % S].transpose(1, 2).float().contiguous()


def _scores(q, k, seen):
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * q.shape[-1] ** -0.5
    return s.masked_fill(~seen, -math.inf)


def _run_prefix(s, c):
    q, kc, vc, table, lengths = (s[n] for n in ("q", "kc", "vc", "table", "lengths"))
    if own:
        return {"o": _api().paged_prefix_attention(
            q, kc, vc, table, lengths, s["starts"], s["prefix"], enable_gqa=c["Hq"] != c["Hkv"],
            backend="triton")}
    B, Hq, N, D = q.shape
    H, G, n = c["Hkv"], c["G"], c["n_hi"]
    R = Hq // H * N  # rows of a sequence that read one key head
    starts, prefix, lengths = s["starts"].long(), s["prefix"].long(), lengths.long()
    group = (torch.arange(B, device=q.device)[:, None] >= starts[None, 1:]).sum(1)
    rows = q.float().reshape(B, H, R, D)
    last = (lengths[:, None] - N + torch.arange(N, device=q.device)).repeat(1, Hq // H)  # [B, R]
    # the prefixes: rows of all sequences of a group over the pages of its first one
    member = starts[:-1, None] + torch.arange(n, device=q.device)
    real = member < starts[1:, None]
    member = torch.where(real, member, 0)
    key = torch.arange(c["pre_hi"], device=q.device)
    seen = key <= last[member].flatten(1)[:, None, :, None]
    seen = seen & (key < prefix[:, None])[:, None, None, :]
    gq = rows[member].transpose(1, 2).reshape(G, H, n * R, D)
    zero = torch.zeros_like(prefix)
    first_rows = table[starts[:-1]]
    sp = _scores(gq, _rows_of(kc, first_rows, zero, c["pre_hi"]), seen)
    mp = sp.amax(-1, keepdim=True)
    pp = torch.exp(sp - torch.where(mp == -math.inf, 0.0, mp))
    op = torch.matmul(pp, _rows_of(vc, first_rows, zero, c["pre_hi"]))

    def back(t):  # of groups' rows to the sequences'
        t = t.reshape(G, H, n, R, -1).transpose(1, 2)
        return t[group, torch.arange(B, device=q.device) - starts[group]]

    mp, lp, op = back(mp), back(pp.sum(-1, keepdim=True)), back(op)
    # what follows the prefixes, each sequence's own
    key = prefix[group][:, None] + torch.arange(c["hi"], device=q.device)
    seen = key[:, None, None, :] <= last[:, None, :, None]
    ss = _scores(rows, _rows_of(kc, table, prefix[group], c["hi"]), seen)
    m = torch.maximum(mp, ss.amax(-1, keepdim=True))
    m = torch.where(m == -math.inf, 0.0, m)
    ps = torch.exp(ss - m)
    inside = (key < lengths[:, None])[:, None, :, None]
    v = torch.where(inside, _rows_of(vc, table, prefix[group], c["hi"]), 0.0)
    w = torch.exp(mp - m)
    total = ps.sum(-1, keepdim=True) + w * lp
    o = (torch.matmul(ps, v) + w * op) / torch.where(total > 0, total, 1.0)
    return {"o": o.reshape(B, Hq, N, D).to(q.dtype)}


def _run_fork(s, c):
    S, table, shares, free, parents = (c["page"], s["table"], s["shares"], s["free"], s["parents"])
    if own:
        f = _api().paged_cache_fork(table, s["lengths"], parents, free, shares, page_size=S,
                                    free_start=s["start"], backend="triton")
        out = {"lengths": f.lengths, "sources": f.sources, "targets": f.targets, "tokens": f.tokens,
               "start": f.free_start}
    else:
        B, M = table.shape
        old, lengths = table.clone(), s["lengths"].long()
        held, part = (lengths + S - 1) // S, lengths % S
        rows, j = torch.arange(B, device=table.device), torch.arange(M, device=table.device)
        live = parents >= 0
        par = torch.where(live, parents, 0).long()
        children = torch.zeros(B, dtype=torch.int64, device=table.device)
        children.index_add_(0, par, live.long())
        # the child that goes on in the begun page: the row itself, or its first child
        rank = torch.where(live, torch.where(par == rows, -1, rows), B)
        keeper = torch.full((B,), B, dtype=torch.int64, device=table.device)
        keeper = keeper.scatter_reduce(0, par, rank, "amin")
        begun = (j == held[:, None] - 1) & (part > 0)[:, None]
        change = torch.where(begun, children.clamp(max=1)[:, None], children[:, None]) - 1
        change = torch.where((j < held[:, None]) & (old >= 0), change, 0)
        shares.index_add_(0, old.clamp(min=0).flatten(), change.int().flatten())
        # copies take the first free pages
        copies = live & (part[par] > 0) & (rank != keeper[par])
        place = s["start"].long() + torch.cumsum(copies.long(), 0) - 1
        targets = torch.where(copies, free[place.clamp(0, free.shape[0] - 1)], -1)
        last = (held[par] - 1).clamp(min=0)
        sources = torch.where(copies, old[par, last], -1)
        new = torch.where((j < held[par][:, None]) & live[:, None], old[par], old)
        new = torch.where(copies[:, None] & (j == last[:, None]), targets[:, None], new)
        table.copy_(new)
        # the pages that nobody holds go in front of the free ones that are left
        gone = shares < 0
        shares.clamp_(min=0)
        released = gone.sum()
        start = s["start"].long() + copies.sum() - released
        at = torch.where(gone, start + torch.cumsum(gone.long(), 0) - 1, free.shape[0])
        longer = torch.cat((free, free[:1]))
        longer[at] = torch.arange(shares.shape[0], dtype=torch.int32, device=table.device)
        free.copy_(longer[:-1])
        out = {"lengths": torch.where(live, lengths[par], 0).int(), "sources": sources,
               "targets": targets, "tokens": torch.where(copies, part[par], 0).int(),
               "start": start.int()}
    # the program goes on with what the call returns
    s["lengths"], s["start"] = out["lengths"], out["start"]
    return {**out, "table": table, "shares": shares, "free": free}


def _run_copy(s, c):
    if own:
        _api().paged_cache_copy(s["kc"], s["vc"], s["sources"], s["targets"], tokens=s["tokens"],
                                backend="triton")
    else:
        # pairs that name no pages copy the first pair's
        pair = torch.where(s["sources"] >= 0, torch.arange(c["moved"], device="cuda"), 0)
        src, dst = s["sources"].long()[pair], s["targets"].long()[pair]
        for cache in (s["kc"], s["vc"]):
            moved = cache[src]
            if s["tokens"] is not None:
                kept = torch.arange(c["page"], device="cuda") < s["tokens"][pair][:, None]
                moved = torch.where(kept[:, None, :, None], moved, cache[dst])
            cache[dst] = moved
    return {"k": s["kc"], "v": s["vc"]}


def _run_compact(s, c):
    table, shares, free = s["table"], s["shares"], s["free"]
    if own:
        f = _api().paged_cache_compact(table, free, shares, backend="triton")
        return {"table": f.page_table, "free": f.free_pages, "shares": f.page_shares,
                "sources": f.sources, "targets": f.targets, "used": f.used}
    P, F = shares.shape[0], free.shape[0]
    page = torch.arange(P, device=table.device)
    held = torch.ones(P, dtype=torch.bool, device=table.device)
    held[free.long()] = False
    used = held.sum()
    moves, holes = held & (page >= used), ~held & (page < used)
    # the k-th page behind the front takes the k-th free place in it; place F is nobody's
    sources, targets = (torch.full((F + 1,), -1, dtype=torch.int64, device=table.device)
                        for _ in range(2))
    sources[torch.where(moves, torch.cumsum(moves.long(), 0) - 1, F)] = page
    targets[torch.where(holes, torch.cumsum(holes.long(), 0) - 1, F)] = page
    sources, targets = sources[:F], targets[:F]
    taken = sources >= 0
    place = torch.cat((page, page[:1]))
    place[torch.where(taken, sources, P)] = targets
    place = place[:P]
    new_shares = torch.where(page < used, shares, 0)
    new_shares = torch.cat((new_shares, new_shares[:1]))
    new_shares[torch.where(taken, targets, P)] = shares[sources.clamp(min=0)]
    new_free = used + torch.arange(F, device=table.device)
    return {"table": torch.where(table >= 0, place[table.clamp(min=0).long()], table).int(),
            "free": torch.where(new_free < P, new_free, -1).int(), "shares": new_shares[:P],
            "sources": sources.int(), "targets": targets.int(), "used": used.reshape(1).int()}


_RUN = {"prefix": _run_prefix, "fork": _run_fork, "copy": _run_copy, "compact": _run_compact}


def run(state):
    return _RUN[state["case"]["op"]](state, state["case"])


# ---- what a pass cannot do without ------------------------------------------------------


def work(case):
    op = case["op"]
    if op == "copy":
        pairs = case["moved"] - case["moved"] // 8
        tokens = case["page"] / 2 if case["part"] else case["page"]
        values = int(pairs * tokens) * case["Hkv"] * case["D"]
        return {"bytes": 8 * values + 8 * case["moved"], "flops": 0}
    n, pre, lengths = _sizes(case)
    B, S = sum(n), case["page"]
    if op == "prefix":
        own_keys = sum(lengths) - sum(p * k for p, k in zip(pre, n))
        q = B * case["Hq"] * case["N"] * case["D"]
        keys = sum(pre) + own_keys
        return {"bytes": 4 * q + 4 * keys * case["Hkv"] * case["D"] + 4 * keys // S,
                "flops": 4 * sum(lengths) * case["Hq"] * case["N"] * case["D"]}
    entries = sum(_cdiv(x, S) for x in lengths)
    if op == "fork":
        # a row's entries read and written, a count for each page that changes hands
        return {"bytes": 16 * entries + 32 * B, "flops": 2 * entries}
    used = _used_pages(case)
    pages = used + max(1, int(used * (1 / case["held"] - 1)))
    # the table and the counts read and written, the free pages read, and written with the moves
    return {"bytes": 8 * entries + 8 * pages + 16 * (pages - used), "flops": 4 * pages}


# ---- the definitions in 64 bits ---------------------------------------------------------


def _exact_prefix(s, c):
    B, Hq, N, D = s["q"].shape
    H, S = c["Hkv"], c["page"]
    n, pre, lengths = _sizes(c)
    table, rows, b = s["table"].long(), Hq // H, 0
    out = torch.zeros(B, Hq, N, D, dtype=torch.float64, device="cuda")
    for size, shared in zip(n, pre):
        at = torch.arange(shared, device="cuda")
        front = [[t[table[b][at // S], h, at % S].double() for t in (s["kc"], s["vc"])]
                 for h in range(H)]
        for i in range(b, b + size):
            at = torch.arange(shared, lengths[i], device="cuda")
            page = table[i][at // S]
            for h in range(H):
                k, v = (torch.cat((f, t[page, h, at % S].double()))
                        for f, t in zip(front[h], (s["kc"], s["vc"])))
                heads = slice(h * rows, (h + 1) * rows)
                for e in range(N):
                    seen = lengths[i] - N + e + 1
                    score = s["q"][i, heads, e].double() @ k[:seen].t() / math.sqrt(D)
                    p = torch.softmax(score, -1)
                    out[i, heads, e] = p @ v[:seen]
        b += size
    return {"o": out}


def _exact_fork(s, c):
    S, table, start = c["page"], s["table"].tolist(), int(s["start"])
    free, lengths, parents = (s[n].tolist() for n in ("free", "lengths", "parents"))
    B, holders = len(table), {}
    before = [row[:_cdiv(x, S)] for row, x in zip(table, lengths)]
    sources, targets, tokens, after, new = [-1] * B, [-1] * B, [0] * B, [], []
    claimed = {p: p for p in parents if p >= 0 and parents[p] == p}
    for b, p in enumerate(parents):
        row = list(before[p]) if p >= 0 else []
        if p >= 0 and lengths[p] % S and claimed.setdefault(p, b) != b:
            sources[b], targets[b], tokens[b] = row[-1], free[start], lengths[p] % S
            row[-1] = free[start]
            start += 1
        after.append(row)
        new.append(lengths[p] if p >= 0 else 0)
    shares = s["shares"].tolist()
    for row in before:
        for page in row:
            holders[page] = holders.get(page, shares[page] + 1) - 1
    for row in after:
        for page in row:
            holders[page] = holders.get(page, 0) + 1
    gone = sorted(page for page, k in holders.items() if k == 0)
    for page, k in holders.items():
        shares[page] = max(k - 1, 0)
    start -= len(gone)
    free[start:start + len(gone)] = gone
    for b, row in enumerate(after):
        table[b][:len(row)] = row
    return {"lengths": _ints(new), "sources": _ints(sources), "targets": _ints(targets),
            "tokens": _ints(tokens), "start": _ints([start]), "table": _ints(table),
            "shares": _ints(shares), "free": _ints(free)}


def _exact_copy(s, c):
    out = {}
    for n, cache in (("k", s["kc"]), ("v", s["vc"])):
        t = cache.double()
        kept = s["sources"] >= 0
        src, dst = s["sources"][kept].long(), s["targets"][kept].long()
        count = torch.full_like(src, c["page"]) if s["tokens"] is None else s["tokens"][kept].long()
        for r in range(c["page"]):
            t[dst[count > r], :, r] = cache[src[count > r], :, r].double()
        out[n] = t
    return out


def _exact_compact(s, c):
    shares, free = s["shares"].tolist(), s["free"].tolist()
    P, gone = len(shares), set(free)
    used = P - len(gone)
    holes = [p for p in range(used) if p in gone]
    moves = [p for p in range(used, P) if p not in gone]
    place = torch.arange(P)
    for a, b in zip(moves, holes):
        place[a] = b
        shares[b] = shares[a]
    pad = [-1] * (len(free) - len(moves))
    table = s["table"].cpu()
    table = torch.where(table >= 0, place[table.clamp(min=0).long()].int(), table)
    new = list(range(used, P))
    return {"table": table.cuda(), "free": _ints(new + [-1] * (len(free) - len(new))),
            "shares": _ints([x if p < used else 0 for p, x in enumerate(shares)]),
            "sources": _ints(moves + pad), "targets": _ints(holes + pad), "used": _ints([used])}


_EXACT = {"prefix": _exact_prefix, "fork": _exact_fork, "copy": _exact_copy,
          "compact": _exact_compact}


def exact(case, seed):
    # The small steps of the 64-bit form take about a millisecond: many of them are left out.
    if case["op"] == "prefix" and sum(_sizes(case)[0]) * case["Hkv"] * case["N"] > 8000:
        return None
    return _EXACT[case["op"]](prepare(case, seed), case)
