"""Counts of pages, forks, room and compaction, entry by entry from the definitions, in plain Python."""


class PlainPages:
    """`table`: a list of lists.  `copied`: the (source, place) pairs of the last call."""

    def __init__(self, pages, page_size):
        self.pages, self.page, self.refs, self.copied, self.missing, self.used = pages, page_size, [0] * pages, [], 0, 0

    def is_page(self, q):
        return 0 <= q < self.pages

    def fork(self, table, lens, parents, width=None):
        out = []
        for b in parents:
            row = []
            for j in range(len(table[0]) if width is None else width):
                q = table[b][j] if 0 <= b < len(table) and j < len(table[b]) and (lens is None or j * self.page < lens[b]) else -1
                row.append(q if self.is_page(q) else -1)
                if row[-1] >= 0:
                    self.refs[q] += 1
            out.append(row)
        return out

    def free(self, table, lens=None):
        for b, row in enumerate(table):
            for j, q in enumerate(row):
                if lens is None or j * self.page >= max(lens[b], 0):
                    row[j] = -1
                    if self.is_page(q) and self.refs[q] > 0:
                        self.refs[q] -= 1

    def extend(self, table, lens, more):
        self.copied, self.missing = [], 0
        at = []
        for b, row in enumerate(table):
            n, m = max(lens[b], 0), more[b]
            at += [(b, j) for j in range(n // self.page, min(-(-(n + m) // self.page), len(row))) if m >= 0]
        holders = {}
        for b, j in at:
            q = table[b][j]
            if self.is_page(q) and self.refs[q] > 1:
                holders.setdefault(q, []).append((b, j))
        keeps = {who[0] for q, who in holders.items() if len(who) == self.refs[q]}
        gives = {x for who in holders.values() for x in who if x not in keeps}
        take = [(b, j) for b, j in at if not self.is_page(table[b][j]) or (b, j) in gives]
        free = [p for p in range(self.pages) if self.refs[p] == 0]
        if len(take) > len(free):
            self.missing = len(take) - len(free)
            for b, j in at:
                if not self.is_page(table[b][j]):
                    table[b][j] = -1
            return
        for (b, j), p in zip(take, free):
            q = table[b][j]
            if (b, j) in gives:
                self.refs[q] -= 1
                self.copied.append((q, p))
            table[b][j], self.refs[p] = p, 1

    def compact(self, *tables):
        live = [p for p in range(self.pages) if self.refs[p] > 0]
        self.used = n = len(live)
        self.copied = list(zip([p for p in live if p >= n], [p for p in range(n) if self.refs[p] <= 0]))
        to = {p: p for p in live} | dict(self.copied)
        for src, dst in self.copied:
            self.refs[dst], self.refs[src] = self.refs[src], 0
        for table in tables:
            for row in table:
                for j, q in enumerate(row):
                    if self.is_page(q):
                        row[j] = to.get(q, -1)
