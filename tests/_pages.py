"""Requests that share pages, one after another in Python: what fork, free and compact
are to leave behind."""


def pages_of(n, page):
    return -(-n // page)


class Pool:
    def __init__(self, num_pages, rows, width, free=None):
        self.rows = [[-1] * width for _ in range(rows)]
        self.shared = [0] * num_pages
        self.free = list(range(num_pages)) if free is None else list(free)
        self.head = 0

    def take(self, row, n):
        """What build_page_tables does: n more pages for a row."""
        have = sum(x >= 0 for x in self.rows[row])
        for j in range(have, have + n):
            self.rows[row][j] = self.free[self.head]
            self.head += 1

    def fork(self, parents, children, lens, page):
        src, dst = [], []
        taken = set(children)
        seen = set()
        for p, c, n in zip(parents, children, lens):
            s = d = -1
            if (c not in seen and p not in taken and 0 <= c < len(self.rows) and 0 <= p < len(self.rows)
                    and 0 <= n <= page * len(self.rows[0])):
                full = n // page
                for j in range(full):
                    self.rows[c][j] = self.rows[p][j]
                    self.shared[self.rows[p][j]] += 1
                if n % page:
                    if self.head < len(self.free):
                        s, d = self.rows[p][full], self.free[self.head]
                    self.rows[c][full] = d
                    self.head = min(self.head + 1, len(self.free))
            seen.add(c)
            src.append(s)
            dst.append(d)
        return src, dst

    def give_back(self, rows, lens, page):
        """Free: a page goes back at its last entry of the call."""
        freed, seen = [], set()
        for r, n in zip(rows, lens):
            if r in seen or not 0 <= r < len(self.rows) or not 0 <= n <= page * len(self.rows[0]):
                continue
            seen.add(r)
            for j in range(pages_of(n, page)):
                p = self.rows[r][j]
                self.rows[r][j] = -1
                if p < 0:
                    continue
                if self.shared[p] > 0:
                    self.shared[p] -= 1
                else:
                    freed.append(p)
        self.head -= len(freed)
        self.free[self.head:self.head + len(freed)] = freed

    def compact(self, rows, lens, page, max_moves):
        held = {}
        for r, n in zip(rows, lens):
            for j in range(pages_of(n, page)):
                held.setdefault(self.rows[r][j], []).append((r, j))
        L = len(held)
        movers = sorted((p for p in held if p >= L), reverse=True)[:max_moves]
        holes = [p for p in range(L) if p not in held][:len(movers)]
        for s, d in zip(movers, holes):
            for r, j in held[s]:
                self.rows[r][j] = d
            self.shared[d], self.shared[s] = self.shared[s], 0
        live = (set(held) - set(movers)) | set(holes)
        rest = [p for p in range(len(self.shared)) if p not in live]
        self.free[len(self.free) - len(rest):] = rest
        self.head = len(self.free) - len(rest)
        pad = [-1] * (max_moves - len(movers))
        return movers + pad, holes + pad
