"""Page allocation, sharing and compaction restated on Python lists (test infrastructure
only; the reference hands pages out on the host and shares none, so there is no golden
vector)."""
from __future__ import annotations

PS = 16


class Pages:
    """Tables, lengths and counts as lists; ``copied`` collects the (src, dst) page copies."""

    def __init__(self, table, valid, refs):
        self.table = [[list(map(int, r)) for r in s] for s in table]
        self.valid = [list(map(int, s)) for s in valid]
        self.refs = list(map(int, refs))
        self.copied = []

    @property
    def width(self):
        return len(self.table[0][0])

    def used(self, b, h):
        return min(max(0, -(-self.valid[b][h] // PS)), self.width)

    def _in(self, page):
        return 0 <= page < len(self.refs)

    def _free(self):
        return [i for i, r in enumerate(self.refs) if r <= 0]

    def free(self, seqs, tokens=None):
        for k, s in enumerate(seqs):
            if not 0 <= s < len(self.table):
                continue
            for h, row in enumerate(self.table[s]):
                last = self.used(s, h)
                drop = self.valid[s][h] if tokens is None else max(0, tokens[k])
                self.valid[s][h] = max(0, self.valid[s][h] - drop)
                for e in range(self.used(s, h), last):
                    if self._in(row[e]):
                        self.refs[row[e]] -= 1
                    row[e] = -1

    def _sound(self, seqs):
        return all(0 <= s < len(self.table) for s in seqs) and len(set(seqs)) == len(seqs)

    def grow(self, seqs, new, pools=False):
        """``pools``: there are arrays to copy a last page in that others hold too."""
        if not self._sound(seqs) or any(n < 0 for n in new):
            return -1
        needs, shared = [], []
        for s, n in zip(seqs, new):
            for h in range(len(self.table[s])):
                old = max(0, self.valid[s][h])
                if old + n > self.width * PS:
                    return -1
                last = self.table[s][h][old // PS] if n > 0 and old % PS else -1
                anew = self._in(last) and self.refs[last] > 1
                if anew and not pools:
                    return -1
                needs.append((s, h, -(-old // PS) - anew, -(-(old + n) // PS), old + n))
                if anew:
                    shared.append((s, h, old // PS))
        free = self._free()
        need = sum(b - a for _, _, a, b, _ in needs)
        if need > len(free):
            return need - len(free)
        it = iter(free)
        lost = {(s, h): self.table[s][h][e] for s, h, e in shared}
        for page in lost.values():
            self.refs[page] -= 1
        for s, h, a, b, tokens in needs:
            for e in range(a, b):
                self.table[s][h][e] = page = next(it)
                self.refs[page] = 1
            if (s, h) in lost:
                self.copied.append((lost[s, h], self.table[s][h][a]))
            self.valid[s][h] = tokens
        return 0

    def fork(self, parents, children):
        if not self._sound(children) or not all(0 <= p < len(self.table) for p in parents):
            return -1
        if set(parents) & set(children) or any(v for c in children for v in self.valid[c]):
            return -1
        plan = []
        for p, c in zip(parents, children):
            for h in range(len(self.table[p])):
                n = self.used(p, h)
                own = n > 0 and n * PS > self.valid[p][h] and self._in(self.table[p][h][n - 1])
                plan.append((p, c, h, n, own))
        free = self._free()
        need = sum(x[4] for x in plan)
        if need > len(free):
            return need - len(free)
        it = iter(free)
        for p, c, h, n, own in plan:
            row = self.table[c][h]
            row[:n] = self.table[p][h][:n]
            if own:
                page = next(it)
                self.copied.append((row[n - 1], page))
                row[n - 1] = page
            for e in range(n):
                if self._in(row[e]):
                    self.refs[row[e]] += 1
            if own:
                self.refs[row[n - 1]] = 1
            self.valid[c][h] = self.valid[p][h]
        return 0

    def compact(self):
        """(table, refs, page_map, moves); the state itself stays as it is."""
        live = [i for i, r in enumerate(self.refs) if r > 0]
        holes = [i for i in range(len(live)) if self.refs[i] <= 0]
        moves = list(zip(reversed(live), holes))
        to = [i if r > 0 else -1 for i, r in enumerate(self.refs)]
        for s, d in moves:
            to[s] = d
        refs = [0] * len(self.refs)
        for i in live:
            refs[to[i]] = self.refs[i]
        table = [[list(r) for r in s] for s in self.table]
        for b, s in enumerate(table):
            for h, row in enumerate(s):
                for e in range(self.used(b, h)):
                    if self._in(row[e]):
                        row[e] = to[row[e]]
        return table, refs, to, moves
