"""The cache's page operations on the host, one row and one page at a time: what the device calls
(enx_pages_*) have to give, entry for entry."""

NONE_FREE, BAD_LIST = 1, 2


class Pages:
    def __init__(self, rows, width, pages, page_tokens):
        self.table = [[-1] * width for _ in range(rows)]
        self.lengths = [0] * rows
        self.refs = [0] * pages
        self.page = page_tokens
        self.status = 0

    def _held(self, tokens):
        return -(-tokens // self.page)

    def _rows_ok(self, rows):
        return len(set(rows)) == len(rows) and all(0 <= r < len(self.table) for r in rows)

    def free(self, rows, keep):
        if not self._rows_ok(rows) or min(keep, default=0) < 0:
            self.status |= BAD_LIST
            return
        for r, k in zip(rows, keep):
            k = min(k, self.lengths[r])
            for i in range(self._held(k), self._held(self.lengths[r])):
                self.refs[self.table[r][i]] -= 1
                self.table[r][i] = -1
            self.lengths[r] = k

    def fork(self, src, dst):
        if (not self._rows_ok(dst) or not all(0 <= s < len(self.table) for s in src) or set(src) & set(dst)
                or any(self.lengths[d] for d in dst)):
            self.status |= BAD_LIST
            return
        for s, d in zip(src, dst):
            for i in range(self._held(self.lengths[s])):
                self.table[d][i] = self.table[s][i]
                self.refs[self.table[s][i]] += 1
            self.lengths[d] = self.lengths[s]

    def grow(self, rows, add):
        """(pairs, pages taken); ([], 0) when refused."""
        width = len(self.table[0])
        if (not self._rows_ok(rows) or min(add, default=0) < 0
                or any(self.lengths[r] + a > width * self.page for r, a in zip(rows, add))):
            self.status |= BAD_LIST
            return [], 0
        writers = {}
        for r, a in zip(rows, add):
            n = self.lengths[r]
            if a and n % self.page:
                writers.setdefault(self.table[r][n // self.page], []).append(r)
        copies = {r for p, who in writers.items() for r in who
                  if self.refs[p] > 1 and not (len(who) == self.refs[p] and who[0] == r)}
        want = [(r in copies) + self._held(self.lengths[r] + a) - self._held(self.lengths[r]) for r, a in zip(rows, add)]
        free = [p for p, n in enumerate(self.refs) if n == 0][: sum(want)]
        if len(free) < sum(want):
            self.status |= NONE_FREE
            return [], 0
        pairs, at = [], iter(free)
        for r, a in zip(rows, add):
            n = self.lengths[r]
            if r in copies:
                old, new = self.table[r][n // self.page], next(at)
                self.refs[old] -= 1
                self.refs[new] = 1
                self.table[r][n // self.page] = new
                pairs.append((old, new))
            for i in range(self._held(n), self._held(n + a)):
                self.table[r][i] = next(at)
                self.refs[self.table[r][i]] = 1
            self.lengths[r] = n + a
        return pairs, sum(want)

    def compact(self):
        """(pairs, pages in use); the table and the counts take the new numbers."""
        used = [p for p, n in enumerate(self.refs) if n > 0]
        holes = [p for p in range(len(used)) if self.refs[p] == 0]
        movers = [p for p in used if p >= len(used)]
        to = dict(zip(movers, holes))
        for r, row in enumerate(self.table):
            held = self._held(self.lengths[r])
            self.table[r] = [to.get(p, p) if i < held else -1 for i, p in enumerate(row)]
        refs = [0] * len(self.refs)
        for p in used:
            refs[to.get(p, p)] = self.refs[p]
        self.refs = refs
        return list(zip(movers, holes)), len(used)
