"""How the attention over shared prefixes divides its work: the walk of every work-group of
prefix_fwd_kernel (csrc/fa_prefix.hip) over the line of units and the pieces of long prefixes, on the
CPU. Every unit of every tile has to be taken once, into a slot of its own inside the workspace, and the
join has to look where it was written. test_prefix_work.py compares the places with the kernel's."""

from __future__ import annotations

import random
from bisect import bisect_right

import pytest
from test_paged import cdiv

TILE, OWN_ROWS, OWN_TILE, LEAD, OWN_LEAD, LEAST, WAVES = 128, 64, 32, 6, 1, 4, 4  # fa_layer.hpp


def units_of(first, end):
    """Units of 32 keys that the keys first .. end - 1 take; the first begins at a multiple of 16."""
    return cdiv(end - (first & ~15), 32) if end > first else 0


class Line:
    """The division of a call: groups of ``sizes`` sequences, the lengths of all, ``R`` query rows a
    key/value head and ``keys`` that a row of the page table holds."""

    def __init__(self, sizes, prefix, lengths, Hkv, R, D, keys):
        self.B, self.G, self.Hkv, self.R = len(lengths), len(sizes), Hkv, R
        self.waves = R <= OWN_ROWS
        self.starts = [sum(sizes[:g]) for g in range(self.G + 1)]
        self.own_tile, self.lead = (OWN_TILE, OWN_LEAD) if self.waves else (TILE, LEAD)
        self.blocks = cdiv(R, self.own_tile)
        self.HB = Hkv * self.blocks
        # the launch
        groups, own = min(self.G, self.B // 2), self.B * self.HB
        triples = Hkv * (self.B * R // TILE + groups) if groups else 0
        bound = (cdiv(keys, 32) + 1 + LEAD) * (triples + own)
        grid = min(256 * (2 if D > 64 else 3), cdiv(bound, LEAST))
        self.grid = max(cdiv(grid, 8) * 8, 16)
        self.most_pieces = min(self.grid, 256) if self.B * R <= TILE else self.grid
        self.prefix_slots = self.grid + triples if triples else 0
        self.own_slots = WAVES * self.grid + own
        # units of prefixes, and of own keys
        self.front = [min(max(p, 0), lengths[self.starts[g]]) if n > 1 else 0
                      for g, (n, p) in enumerate(zip(sizes, prefix))]
        self.triples = [cdiv(n * R, TILE) * Hkv for n in sizes]
        self.group = []
        for b in range(self.B):
            g = bisect_right(self.starts, b) - 1
            self.group.append(g if 0 <= g < self.G else -1)
        self.own_units = [units_of(self.front[g] if g >= 0 else 0, n)
                          for g, n in zip(self.group, lengths)]
        self.units = [units_of(0, f) for f in self.front]
        self.divide()

    def on_line(self, units, lead):
        return units + lead if units else 0

    def divide(self):
        """prefix_find: the stretches, and the long prefixes' pieces."""
        self.own_all = sum(self.on_line(u, self.lead) * self.HB for u in self.own_units)
        every = sum(self.on_line(u, LEAD) * t for u, t in zip(self.units, self.triples))
        cost = self.own_all - self.own_all // 5 if self.waves else self.own_all
        self.L = L = max(cdiv(every + cost, self.grid - 2), LEAST)
        self.own_stretch = max((5 * L + 15) // 16, 2) if self.waves else L
        is_long = [L >= 2 * LEAD and u >= 2 * (L - LEAD) for u in self.units]
        self.given_up = False
        while True:
            cut = [x and not self.given_up for x in is_long]
            self.on = sum(self.on_line(u, LEAD) * t
                          for u, t, c in zip(self.units, self.triples, cut) if not c)
            long_units = sum(u * t for u, t, c in zip(self.units, self.triples, cut) if c)
            self.cuts = [0] * self.G
            if not long_units:
                break
            rest = (cdiv(self.on, L) + cdiv(self.own_all, WAVES * self.own_stretch) if self.waves
                    else cdiv(self.on + self.own_all, L))
            budget = min(self.grid - rest, self.most_pieces) // 8 * 8
            self.cuts = [max(1, min(int(u * budget / long_units), u // 16)) if c else 0
                         for u, c in zip(self.units, cut)]
            if cdiv(sum(c * t for c, t in zip(self.cuts, self.triples)), 8) * 8 <= self.grid - rest:
                break
            self.given_up = True
        self.pieces = sum(c * t for c, t in zip(self.cuts, self.triples))
        # the join's places, as the kernel leaves them in the workspace
        self.groups, piece, base, first = [], 0, 0, 0
        for u, t, k in zip(self.units, self.triples, self.cuts):
            self.groups.append((piece if k else base, u, first, t // self.Hkv, k))
            if k:
                piece += t * k
            elif u:
                base += self.on_line(u, LEAD) * t
                first += t
        self.seqs, base = [], 0 if self.waves else self.on
        for b, (g, u) in enumerate(zip(self.group, self.own_units)):
            self.seqs.append((base, u, g, b - self.starts[g] if g >= 0 else 0))
            base += self.on_line(u, self.lead) * self.HB

    def triples_on_line(self):
        """(kind, group or sequence, triple of it, its first place, units, lead, triple of the line)."""
        for g, (base, u, first, _, k) in enumerate(self.groups):
            if u and not k:
                for sub in range(self.triples[g]):
                    yield "prefix", g, sub, base + sub * (u + LEAD), u, LEAD, first + sub
        yield from () if self.waves else self.own_triples()

    def own_triples(self):
        for b, (base, u, _, _) in enumerate(self.seqs):
            if u:
                for sub in range(self.HB):
                    yield "own", b, sub, base + sub * (u + self.lead), u, self.lead, b * self.HB + sub

    def walk(self):
        """(kind, group or sequence, triple of it, units taken, slot) of all pieces."""
        def stretches(triples, length):
            for kind, at, sub, place, u, lead, t in triples:
                for s in range(place // length, cdiv(place + lead + u, length)):
                    u0 = max(s * length - place - lead, 0)
                    u1 = min(max((s + 1) * length - place - lead, 0), u)
                    if u1 > u0:
                        yield s, (kind, at, sub, u0, u1,
                                  s + t + (self.pieces if kind == "prefix" else 0))
        lines = [(self.on if self.waves else self.on + self.own_all, self.L, self.triples_on_line())]
        if self.waves:
            lines.append((self.own_all, self.own_stretch, self.own_triples()))
        taken = [{} for _ in lines]
        for to, (_, length, triples) in zip(taken, lines):
            for s, piece in stretches(triples, length):
                to.setdefault(s, []).append(piece)
        each, on = cdiv(self.pieces, 8), cdiv(self.on, self.L) if self.waves else 0
        done = []
        for block in range(self.grid):
            xcd, i = block % 8, block // 8
            if i < each:
                if xcd * each + i < self.pieces:
                    done.append(self.piece(xcd * each + i))
                continue
            s = (i - each) * 8 + xcd
            if self.waves and s >= on:
                for w in range(WAVES):
                    done += taken[1].pop((s - on) * WAVES + w, [])
            else:
                done += taken[0].pop(s, [])
        assert not any(taken), "stretches that no work-group takes"
        return done

    def piece(self, s):
        for g, (base, u, _, tiles, k) in enumerate(self.groups):
            if k and base <= s < base + self.triples[g] * k:
                at = s - base
                p = at // tiles % k
                return "prefix", g, at // tiles // k * tiles + at % tiles, u * p // k, u * (p + 1) // k, s
        raise AssertionError("a piece of no group")

    def joined(self, kind, at, sub):
        """Slots of a triple in the order in which the join reads them."""
        def of(base, units, lead, stretch, slot):
            s0 = (base + lead) // stretch
            return [slot + s for s in range(s0, (base + lead + units - 1) // stretch + 1)]
        if kind == "own":
            base, u, _, _ = self.seqs[at]
            return of(base + sub * (u + self.lead), u, self.lead, self.own_stretch, at * self.HB + sub)
        base, u, first, tiles, k = self.groups[at]
        if k:
            return [base + (sub // tiles * k + i) * tiles + sub % tiles for i in range(k)]
        return of(base + sub * (u + LEAD), u, LEAD, self.L, self.pieces + first + sub)


def check_line(*case):
    line = Line(*case)
    done = line.walk()
    for kind, most in (("prefix", line.prefix_slots), ("own", line.own_slots)):
        slots = [d[5] for d in done if d[0] == kind]
        assert len(set(slots)) == len(slots) and all(0 <= s < most for s in slots), kind
    of = {}
    for kind, at, sub, u0, u1, slot in done:
        of.setdefault((kind, at, sub), []).append((u0, u1, slot))
    wanted = [("prefix", g, sub, u) for g, u in enumerate(line.units) if u
              for sub in range(line.triples[g])]
    wanted += [("own", b, sub, u) for b, u in enumerate(line.own_units) if u for sub in range(line.HB)]
    for kind, at, sub, u in wanted:
        parts = sorted(of.pop((kind, at, sub)))
        assert [p[0] for p in parts] == [0] + [p[1] for p in parts[:-1]] and parts[-1][1] == u
        assert [p[2] for p in parts] == line.joined(kind, at, sub)
        assert len(parts) <= line.grid * (WAVES if kind == "own" and line.waves else 1)
    assert not of
    return line


@pytest.mark.parametrize("seed", range(4))
def test_every_unit_is_taken_once(seed):
    rng = random.Random(seed)
    for _ in range(60):
        sizes = [rng.choice([0, 1, 2, 2, 3, 9, 40]) for _ in range(rng.choice([0, 1, 2, 3, 5, 20]))]
        most, own = rng.choice([40, 400, 3000, 20000]), rng.choice([1, 30, 200, 1000])
        prefix = [rng.randint(0, most) for _ in sizes]
        lengths = [max(0, p + rng.randint(-5, own)) for n, p in zip(sizes, prefix) for _ in range(n)]
        lengths += [rng.randint(0, own) for _ in range(rng.choice([0, 3, 60]) or not lengths)]
        keys = cdiv(max([1, *lengths]), 16) * 16 * rng.choice([1, 1, 3])
        check_line(sizes, prefix, lengths, rng.choice([1, 2, 8]), rng.choice([1, 4, 16, 33, 64, 66, 200]),
                   rng.choice([32, 64, 128]), keys)


@pytest.mark.parametrize("R", [8, 64, 100, 120])
def test_every_unit_is_taken_once_near_the_room_for_pieces(R):
    """Own keys that leave the long prefixes some work-groups, or too few for their pieces, which come
    in eights: all three outcomes have to occur."""
    rng = random.Random(R)
    seen = set()
    blocks = cdiv(R, OWN_TILE if R <= OWN_ROWS else TILE)
    for _ in range(150):
        n, L = rng.choice([1, 2, 3, 9, 10, 17, 30]), rng.randint(12, 20)
        units = max(2 * (L - LEAD) + rng.choice([-1, 0, 1, 2, 20]), 1)
        sizes = [2] * n
        triples = n * cdiv(2 * R, TILE)
        target = 510 * L - triples * (units + LEAD)  # what the own keys have to cost
        if R <= OWN_ROWS:
            target += target // 4
        own, total = [], 0
        while total < target:
            own.append(rng.randint(20, 120))
            total += (own[-1] + (OWN_LEAD if R <= OWN_ROWS else LEAD)) * blocks
        if rng.random() < 0.7:  # as near as can be below it
            own[-1] = max(1, own[-1] - cdiv(total - target, blocks))
        line = check_line(sizes, [32 * units] * n, [32 * units] * sum(sizes) + [32 * u for u in own], 1, R,
                          128, 120 * 32)
        seen.add("given up" if line.given_up else "pieces" if line.pieces else "none")
    assert seen == {"given up", "pieces", "none"}
