"""Plain forms of what the batched decoding operators do at their edges, from the header's words."""
import decoding_ref as D


class SharedPool(D.Pool):
    """A pool whose rows may share any page.  The one that goes on with a source's own pages takes the partial last one
    only where no other row holds it, and those behind up to the first that another row holds."""

    def fork(self, src):
        n, free = len(self.rows), self.free_pages()
        keeper = {}
        for i, r in enumerate(src):
            if 0 <= r < n and (r not in keeper or r == i):
                keeper[r] = i
        rows, lens, copies, lacked = [], [], [], 0
        for i, r in enumerate(src):
            if not 0 <= r < n:
                rows.append([])
                lens.append(0)
                continue
            full, touched = self.size(r)
            old = self.rows[r]
            row = old[:touched]
            alone = [not self.known(p) or self.refs[p] == 1 for p in old]
            if keeper[r] == i:
                for p, a in zip(old[touched:], alone[touched:]):
                    if not a:
                        break
                    row.append(p)
            if touched > full and len(old) > full and (keeper[r] != i or not alone[full]):
                row[full] = free.pop(0) if free else -1
                lacked += row[full] < 0
                if row[full] >= 0 and self.known(old[full]):
                    copies.append((old[full], row[full]))
            rows.append(row)
            lens.append(self.lens[r])
        for p in (p for r in self.rows for p in r if self.known(p)):
            self.refs[p] -= 1
        for p in (p for r in rows for p in r if self.known(p)):
            self.refs[p] += 1
        for c in self.caches:
            for a, b in copies:
                c[b] = c[a]
        self.rows, self.lens, self.counts[0] = rows, lens, lacked

    def reserve(self):
        super().reserve()
        self.counts[0] += sum(max(0, -(-x // self.page) - self.cols) for x in self.lens)
