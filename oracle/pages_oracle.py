"""Pages of a cache restated in plain Python, one sequence after the other: what each has, which are free, what is copied."""
import numpy as np


class Pages:
    def __init__(self, table, lengths, uses, page):
        self.page, self.width = page, table.shape[1]
        self.lengths, self.uses = [int(n) for n in lengths], [int(n) for n in uses]
        self.rows = [[int(x) for x in row[:self.count(n)]] for row, n in zip(table, lengths)]
        self.missing = 0

    def count(self, tokens):
        return -(-int(tokens) // self.page)

    def table(self):
        return np.array([row + [-1] * (self.width - len(row)) for row in self.rows], dtype=np.int32)

    def state(self):
        return self.table(), np.array(self.lengths, dtype=np.int32), np.array(self.uses, dtype=np.int32)

    def free_pages(self):
        return [p for p, n in enumerate(self.uses) if n == 0]

    def append(self, offsets, tokens):
        slots, free, promised = [-1] * tokens, self.free_pages(), 0
        for b in range(len(self.rows)):
            new = max(0, offsets[b + 1] - offsets[b])
            total = self.lengths[b] + new
            need = self.count(total) - len(self.rows[b])
            if self.count(total) > self.width:
                self.missing += 1
                continue
            promised += need                          # those in front of it come first, whether they got theirs or not
            if need and promised > len(free):
                self.missing += 1
                continue
            taken = free[promised - need:promised]
            for p in taken:
                self.uses[p] = 1
            self.rows[b] += taken
            for i in range(new):
                at = self.lengths[b] + i
                slots[offsets[b] + i] = self.rows[b][at // self.page] * self.page + at % self.page
            self.lengths[b] = total
        return np.array(slots, dtype=np.int32)

    def free(self, which):
        for b in which:
            if 0 <= b < len(self.rows):
                for p in self.rows[b]:
                    self.uses[p] -= 1
                self.rows[b], self.lengths[b] = [], 0

    def fork(self, parents, children):
        count, known = len(parents), range(len(self.rows))
        sources, targets, seen, valid = [-1] * count, [-1] * count, set(), []
        for i, (a, c) in enumerate(zip(parents, children)):
            if a in known and c in known and c not in seen:
                seen.add(c)
                valid.append(i)
        rows, lengths = [list(r) for r in self.rows], list(self.lengths)
        for c in seen:
            for p in rows[c]:
                self.uses[p] -= 1
        heirs, copying = set(), []
        for i in valid:
            a, c = parents[i], children[i]
            self.rows[c], self.lengths[c] = list(rows[a]), lengths[a]
            partial = lengths[a] % self.page != 0
            copied = partial and (a not in seen or a in heirs)
            heirs.add(a)
            for p in rows[a][:len(rows[a]) - copied]:
                self.uses[p] += 1
            if copied:
                copying.append(i)
        free = self.free_pages()
        for rank, i in enumerate(copying):
            c = children[i]
            if rank < len(free):
                sources[i], targets[i] = self.rows[c][-1], free[rank]
                self.rows[c][-1] = free[rank]
                self.uses[free[rank]] = 1
            else:
                for p in self.rows[c][:-1]:
                    self.uses[p] -= 1
                self.rows[c], self.lengths[c] = [], 0
                self.missing += 1
        return np.array(sources, dtype=np.int32), np.array(targets, dtype=np.int32)

    def compact(self):
        used = sum(1 for n in self.uses if n > 0)
        targets = [p for p in range(used) if self.uses[p] == 0]
        sources = [p for p in range(used, len(self.uses)) if self.uses[p] > 0]
        to = dict(zip(sources, targets))
        self.rows = [[to.get(p, p) for p in row] for row in self.rows]
        for a, b in to.items():
            self.uses[b], self.uses[a] = self.uses[a], 0
        rest = [-1] * (len(self.uses) // 2 - len(sources))
        return np.array(sources + rest, dtype=np.int32), np.array(targets + rest, dtype=np.int32)

    def check(self):
        """What holds between calls: uses count the rows, a last page that is not full belongs to one."""
        counted = [0] * len(self.uses)
        for row, n in zip(self.rows, self.lengths):
            assert len(row) == self.count(n) and len(set(row)) == len(row)
            for p in row:
                counted[p] += 1
        assert counted == self.uses
        for row, n in zip(self.rows, self.lengths):
            if n % self.page:
                assert self.uses[row[-1]] == 1
