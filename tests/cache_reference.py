"""What becomes of a paged cache's books when requests go on from others, end, or move: the definition, step by step on the host."""


class Books:
    """Lists of a cache's numbers: tables (a list of pages a request), lengths, the free pages in their order, and what each page holds (any value a slot)."""

    def __init__(self, pages, page, batch, width):
        self.pages, self.page, self.width = pages, page, width
        self.tables = [[] for _ in range(batch)]
        self.lengths = [0] * batch
        self.free = list(range(pages))
        self.slots = {}

    def append(self, new):
        """new: a list of values for each request."""
        for b, values in enumerate(new):
            for x in values:
                if self.lengths[b] == len(self.tables[b]) * self.page:
                    if not self.free or len(self.tables[b]) == self.width:
                        break
                    self.tables[b].append(self.free.pop(0))
                self.slots[self.tables[b][-1], self.lengths[b] % self.page] = x
                self.lengths[b] += 1

    def values(self, b):
        return [self.slots[self.tables[b][i // self.page], i % self.page] for i in range(self.lengths[b])]

    def shares(self):
        n = [0] * self.pages
        for t in self.tables:
            for p in t:
                n[p] += 1
        return [max(x - 1, 0) for x in n]

    def fork(self, parents):
        batch = len(self.tables)
        parents = [s if 0 <= s < batch else -1 for s in parents]
        old, lengths = [list(t) for t in self.tables], list(self.lengths)
        heir = {}
        for b, s in enumerate(parents):
            if s >= 0:
                heir.setdefault(s, s if parents[s] == s else b)
        kept = {p for s in set(parents) if s >= 0 for p in old[s]}
        for s in range(batch):
            for p in old[s]:
                if p not in kept:
                    kept.add(p)
                    self.free.append(p)
        for b, s in enumerate(parents):
            if s == b:
                continue
            if s < 0:
                self.tables[b], self.lengths[b] = [], 0
                continue
            self.tables[b], self.lengths[b] = list(old[s]), lengths[s]
            rest = lengths[s] % self.page
            if rest and heir[s] != b:
                last = self.tables[b].pop()
                if not self.free:
                    self.lengths[b] -= rest
                    continue
                to = self.free.pop(0)
                for i in range(rest):
                    self.slots[to, i] = self.slots[last, i]
                self.tables[b].append(to)

    def compact(self, room):
        number, slots = {}, {}
        for b, t in enumerate(self.tables):
            for i, p in enumerate(t):
                number.setdefault(p, len(number))
        for b, t in enumerate(self.tables):
            cut = next((i for i, p in enumerate(t) if number[p] >= room), len(t))
            if cut < len(t):
                self.lengths[b] = cut * self.page
            for p in t[:cut]:
                for i in range(self.page):
                    if (p, i) in self.slots:
                        slots[number[p], i] = self.slots[p, i]
            self.tables[b] = [number[p] for p in t[:cut]]
        self.pages, self.slots = room, slots
        self.free = list(range(min(len(number), room), room))
