"""Page tables as a sequential program keeps them, one row after the other."""
from __future__ import annotations


class Tables:
    def __init__(self, rows, lens, managed, n_pages, page_tokens, max_pages):
        self.rows, self.lens = [list(r) for r in rows], list(lens)
        self.managed, self.n_pages, self.P, self.max_pages = sorted(managed), n_pages, page_tokens, max_pages
        self.failed = 0

    def refs(self):
        n = [0] * self.n_pages
        for row in self.rows:
            for p in row:
                n[p] += 1
        return n

    def table(self):
        return [row + [-1] * (self.max_pages - len(row)) for row in self.rows]

    def resize(self, want):
        """Returns the copies made: (from, to, tokens)."""
        for r, n in enumerate(want):
            if 0 <= n < self.lens[r]:
                del self.rows[r][-(-n // self.P):]
                self.lens[r] = n
        refs = self.refs()
        limit = self.max_pages * self.P
        writers = {}
        for r, n in enumerate(want):
            if self.lens[r] < n <= limit and self.lens[r] % self.P and refs[self.rows[r][-1]] > 1:
                writers.setdefault(self.rows[r][-1], []).append(r)
        keeper = {rs[-1] for p, rs in writers.items() if len(rs) == refs[p]}
        shares = {r for rs in writers.values() for r in rs}
        free = [p for p in self.managed if refs[p] == 0]
        asked, copies = 0, []
        for r, n in enumerate(want):
            if n <= self.lens[r]:
                continue
            if n > limit:
                self.failed += 1
                continue
            copy = r in shares and r not in keeper
            need = -(-n // self.P) - len(self.rows[r]) + copy
            asked += need
            if asked > len(free) and (need or r in shares):
                self.failed += 1
                continue
            ids = free[asked - need:asked]
            if copy:
                copies.append((self.rows[r][-1], ids[0], self.lens[r] % self.P))
                self.rows[r][-1] = ids.pop(0)
            self.rows[r] += ids
            self.lens[r] = n
        return copies

    def fork(self, parent):
        rows, lens = [list(r) for r in self.rows], list(self.lens)
        for r, p in enumerate(parent):
            self.failed += p >= len(rows)
            if 0 <= p < len(rows):
                self.rows[r], self.lens[r] = list(rows[p]), lens[p]

    def compact(self):
        """Returns the moves: (from, to)."""
        refs = self.refs()
        used = [p for p in self.managed if refs[p]]
        lowest = self.managed[:len(used)]
        moves = list(zip([p for p in used if p not in set(lowest)], [p for p in lowest if not refs[p]]))
        to = dict(moves)
        self.rows = [[to.get(p, p) for p in row] for row in self.rows]
        return moves
