"""Page tables and pools in numpy, entry by entry, from the operators' definitions."""
import numpy as np


class Tables:
    """tables [sequences][width], lengths, references; pools: arrays [pages][...] and whether a page's slots lie on axis 1 or 2."""

    def __init__(self, tables, lengths, references, page, pools=()):
        self.tables, self.lengths, self.references = (np.array(a, dtype=np.int64) for a in (tables, lengths, references))
        self.page, self.pools = page, [(np.array(p), axis) for p, axis in pools]
        self.missing = 0

    @property
    def pages(self):
        return len(self.references)

    def length(self, b):
        return int(np.clip(self.lengths[b], 0, self.tables.shape[1] * self.page))

    def held(self, b):
        """The entries of a row."""
        return [int(p) for p in self.tables[b, :-(-self.length(b) // self.page)]]

    def inside(self, p):
        return 0 <= p < self.pages

    def free(self):
        return [p for p in range(self.pages) if self.references[p] <= 0]

    def reserve(self, new, capacity):
        slots, positions, free = [], [], self.free()
        lacking, lengths = 0, self.lengths.copy()
        for b, n in enumerate(new):
            n = min(max(int(n), 0), capacity - len(slots))
            length = self.length(b)
            end, out = length, False
            for pos in range(length, length + n):
                slot = where = -1
                if pos < self.tables.shape[1] * self.page:
                    if pos % self.page == 0:
                        if free:
                            p = free.pop(0)
                            self.tables[b, pos // self.page] = p
                            self.references[p] = 1
                        else:
                            lacking, out = lacking + 1, True
                    if not out:
                        p = int(self.tables[b, pos // self.page])
                        slot, where, end = p * self.page + pos % self.page if self.inside(p) else -1, pos, pos + 1
                slots.append(slot)
                positions.append(where)
            lengths[b] = end
        self.lengths, self.missing = lengths, lacking
        rest = capacity - len(slots)
        return np.array(slots + [-1] * rest), np.array(positions + [-1] * rest)

    def trim(self, keep):
        for b, k in enumerate(keep):
            end = min(self.length(b), max(int(k), 0))
            for p in self.held(b)[-(-end // self.page):]:
                if self.inside(p):
                    self.references[p] -= 1
            self.lengths[b] = end

    def fork(self, parents):
        n = len(self.lengths)
        old, lengths = [self.held(b) for b in range(n)], [self.length(b) for b in range(n)]
        children = {x: [b for b in range(n) if parents[b] == x] for x in range(n)}
        rows, copies = {}, []
        for b in range(n):
            p = int(parents[b])
            if p == b:
                continue
            for e in old[b]:
                if self.inside(e):
                    self.references[e] -= 1
            rows[b] = []
            if not 0 <= p < n:
                continue
            rows[b] = list(old[p])
            keeper = p if p in children[p] else children[p][0]
            last = lengths[p] % self.page
            for i, e in enumerate(old[p]):
                if last and i == len(old[p]) - 1 and b != keeper and self.inside(e):
                    copies.append((b, i, e, last))
                elif self.inside(e):
                    self.references[e] += 1
        free = self.free()
        new_lengths = {b: lengths[int(parents[b])] if rows[b] or 0 <= parents[b] < n else 0 for b in rows}
        moved = []
        for b, i, e, last in copies:
            if free:
                rows[b][i] = free.pop(0)
                self.references[rows[b][i]] = 1
                moved.append((e, rows[b][i], last))
            else:
                new_lengths[b] = i * self.page
                rows[b] = rows[b][:i]
        self.missing = len(copies) - len(moved)
        for b, row in rows.items():
            self.tables[b, :len(row)] = row
            self.lengths[b] = new_lengths[b]
        for pool, axis in self.pools:
            for source, target, tokens in moved:
                at = (slice(None),) * (axis - 1) + (slice(0, tokens),)
                pool[target][at] = pool[source][at]

    def compact(self):
        used = [p for p in range(self.pages) if self.references[p] > 0]
        n = len(used)
        movers, holes = [p for p in used if p >= n], [p for p in range(n) if self.references[p] <= 0]
        mapping = np.full(self.pages, -1)
        mapping[used] = used
        for m, h in zip(movers, holes):
            mapping[m] = h
            self.references[h], self.references[m] = self.references[m], 0
            for pool, _ in self.pools:
                pool[h] = pool[m]
        for b in range(len(self.lengths)):
            for i, p in enumerate(self.held(b)):
                if self.inside(p) and mapping[p] >= 0:
                    self.tables[b, i] = mapping[p]
        return mapping, n
