"""Plain forms of what the batched decoding operators do at their edges, from the header's words."""
import math

import torch

import decoding_ref as D
import serving8_ref as R8

MIN, MAX = R8.MIN, R8.MAX


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


def append(codes, scale, table, page, block, first, x):
    """serving8_ref.append with quotients that are rounded once, and scales as the header reads them: from 0 to 2^-60 up
    to it (0 being of zeros), negative and larger ones NaN.  Quotients of f64 numbers of at most 32 bits are next to a
    half only where they are one (they differ from it by 2^-34 at least), so f64 division finds every tie."""
    x = x.double()
    p, L = first, first + x.shape[0]
    while p < L:
        b0 = p // block * block
        e = min(b0 + block, L)
        pg, slot, nb = int(table[p // page]), b0 % page, b0 % page // block
        y = x[p - first:e - first]
        if 0 <= pg < codes.shape[0]:
            for h in range(x.shape[1]):
                was = float(scale[pg, nb, h]) if p > b0 else 0.0
                was = math.nan if not 0 <= was <= MAX else max(was, MIN) if was > 0 else 0.0
                now = float((y[:, h].abs().max() / 127).float())
                now = 0.0 if now < MIN else now
                now = math.nan if not bool(torch.isfinite(y[:, h]).all()) or now > MAX or was != was else max(now, was)
                scale[pg, nb, h] = now
                if now > was and p > b0:
                    old = codes[pg, slot:slot + p - b0, h]
                    codes[pg, slot:slot + p - b0, h] = (old.double() * was / now).round().to(torch.int8)
                at = slice(slot + p - b0, slot + e - b0)
                codes[pg, at, h] = (y[:, h] / now).round().to(torch.int8) if now > 0 else 0
        p = e
