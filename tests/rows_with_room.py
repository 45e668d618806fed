"""Rows with room made ahead: the definition of ``fork_rows`` with ``written``, one row at a
time in Python integers, and what the rows' tokens have to be."""

from __future__ import annotations

import random


class Rows:
    """A block table, its lengths and counts; ``written`` tokens of each row, whose values
    are ``tokens`` (what the row was given) and lie in ``memory`` (by page and slot)."""

    def __init__(self, B, P, N, page):
        self.B, self.P, self.N, self.page = B, P, N, page
        self.table = [[-1] * P for _ in range(B)]
        self.lens, self.refs = [0] * B, [0] * N
        self.tokens = [[] for _ in range(B)]
        self.memory = [[0] * page for _ in range(N)]
        self.next = 1

    @property
    def written(self):
        return [len(t) for t in self.tokens]

    def fork(self, parents=None, new_lens=None, use_written=True):
        """Status and copies (source, destination)."""
        B, page = self.B, self.page
        a = list(range(B)) if parents is None else [p if 0 <= p < B else None for p in parents]
        have = [0 if x is None else self.lens[x] for x in a]
        want = [0 if x is None else h if new_lens is None else max(0, new_lens[b]) for b, (x, h) in enumerate(zip(a, have))]
        if max(want) > self.P * page:
            return 2, []
        reach = [min(h, w) for h, w in zip(have, want)]
        keep = [0 if x is None else min(r, len(self.tokens[x])) if use_written else r for x, r in zip(a, reach)]
        own = lambda p: 0 <= p < self.N and self.refs[p] == 1
        kept = [[] if x is None else self.table[x][:k // page] for x, k in zip(a, keep)]
        heirs = set()
        for x in set(a) - {None}:
            kids = [b for b in range(B) if a[b] == x]
            most = max(keep[b] // page for b in kids)
            kids = [b for b in kids if keep[b] // page == most and -(-reach[b] // page) > most and own(self.table[x][most])]
            if kids:
                heirs.add(x if x in kids else kids[0])
                b = x if x in kids else kids[0]
                for p in self.table[x][most:-(-reach[b] // page)]:
                    if not own(p):
                        break
                    kept[b].append(p)
        heir = [len(kept[b]) > keep[b] // page for b in range(B)]
        free = [p for p, n in enumerate(self.refs) if n == 0]
        copies, table = [], []
        for b in range(B):
            need = -(-want[b] // page) - len(kept[b])
            if need > len(free):
                return 1, []
            if keep[b] % page and not heir[b]:
                copies.append((self.table[a[b]][keep[b] // page], free[0]))
            table.append((kept[b] + free[:need] + [-1] * self.P)[:self.P])
            free = free[need:]
        for sign, rows, lens in ((-1, self.table, self.lens), (1, table, want)):
            for row, n in zip(rows, lens):
                for p in row[:-(-n // page)]:
                    self.refs[p] += sign
        for s, d in copies:
            self.memory[d] = list(self.memory[s])
        self.tokens = [[] if x is None else self.tokens[x][:min(len(self.tokens[x]), w)] for x, w in zip(a, want)]
        self.table, self.lens = table, want
        return 0, copies

    def append(self, b):
        """A new value behind row b's tokens, or 0 where it has no room."""
        n = len(self.tokens[b])
        if n >= self.lens[b]:
            return 0
        self.tokens[b].append(self.next)
        self.memory[self.table[b][n // self.page]][n % self.page] = self.next
        self.next += 1
        return self.next - 1

    def row(self, b):
        """Row b's written tokens as its pages hold them."""
        return [self.memory[self.table[b][n // self.page]][n % self.page] for n in range(len(self.tokens[b]))]


def step(rng: random.Random, m: Rows):
    """The parents and lengths of one random call: rows forked, cut, grown, given room, freed."""
    B, cap = m.B, m.P * m.page
    parents = None if rng.random() < 0.3 else [rng.choice([b, rng.randrange(-1, B + 1)]) for b in range(B)]
    new = None
    if parents is None or rng.random() < 0.6:
        new = []
        for b in range(B):
            a = b if parents is None else parents[b] if 0 <= parents[b] < B else b
            n = len(m.tokens[a])
            new.append(rng.choice([n, n + 1, n + rng.randint(0, 3 * m.page), rng.randint(-1, cap), m.lens[a]]))
        if rng.random() < 0.9:
            new = [min(n, cap) for n in new]
    return parents, new
