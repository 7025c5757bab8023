"""What the calls on a cache's pages do, one after another on the host: the
model that the device's counts, tables, lengths and page contents are compared
with.  A page's content is a label per token slot, None where nothing was
written."""


class Refused(Exception):
    pass


class Pages:
    def __init__(self, pages, seqs, max_pages, page):
        self.page, self.max_pages = page, max_pages
        self.refs = [0] * pages
        self.tables = [[-1] * max_pages for _ in range(seqs)]
        self.lens = [0] * seqs
        self.data = [[None] * page for _ in range(pages)]

    def held(self, n):
        return -(-n // self.page)

    def _free(self, n):
        free = [p for p, r in enumerate(self.refs) if r == 0]
        if len(free) < n:
            raise Refused("too few free pages")
        return free[:n]

    def extend(self, seqs, counts):
        pairs = [(s, c) for s, c in zip(seqs, counts) if s >= 0]
        if any(s >= len(self.lens) for s, _ in pairs):
            raise Refused("outside the cache")
        if len({s for s, _ in pairs}) < len(pairs):
            raise Refused("listed twice")
        if any(c < 0 or self.lens[s] + c > self.max_pages * self.page for s, c in pairs):
            raise Refused("outside the cache")
        new = iter(self._free(sum(self.held(self.lens[s] + c) - self.held(self.lens[s])
                                  for s, c in pairs)))
        for s, c in pairs:
            for j in range(self.held(self.lens[s]), self.held(self.lens[s] + c)):
                p = next(new)
                self.tables[s][j], self.refs[p] = p, 1
            self.lens[s] += c

    def write(self, s, pos, label):
        self.data[self.tables[s][pos // self.page]][pos % self.page] = label

    def read(self, s):
        return [self.data[self.tables[s][t // self.page]][t % self.page]
                for t in range(self.lens[s])]

    def fork(self, parents, children):
        pairs = [(p, c) for p, c in zip(parents, children) if p >= 0 and c >= 0]
        if any(max(p, c) >= len(self.lens) for p, c in pairs):
            raise Refused("outside the cache")
        kids = [c for _, c in pairs]
        if len(set(kids)) < len(kids) or any(self.lens[c] for c in kids) or \
                any(p in kids for p, _ in pairs):
            raise Refused("listed twice")
        new = iter(self._free(sum(self.lens[p] % self.page != 0 for p, _ in pairs)))
        for p, c in pairs:
            full, rest = divmod(self.lens[p], self.page)
            for j in range(full):
                self.tables[c][j] = self.tables[p][j]
                self.refs[self.tables[p][j]] += 1
            if rest:
                q = next(new)
                self.tables[c][full], self.refs[q] = q, 1
                self.data[q][:rest] = self.data[self.tables[p][full]][:rest]
            self.lens[c] = self.lens[p]

    def free(self, seqs):
        for s in seqs:
            if s < 0:
                continue
            for j in range(self.held(self.lens[s])):
                self.refs[self.tables[s][j]] -= 1
            self.lens[s] = 0

    def compact(self):
        used = sum(r > 0 for r in self.refs)
        src = [p for p in range(used, len(self.refs)) if self.refs[p]]
        dst = [p for p in range(used) if not self.refs[p]]
        to = dict(zip(src, dst))
        for a, b in to.items():
            self.data[b] = list(self.data[a])
            self.refs[b], self.refs[a] = self.refs[a], 0
        for s, n in enumerate(self.lens):
            for j in range(self.held(n)):
                self.tables[s][j] = to.get(self.tables[s][j], self.tables[s][j])
