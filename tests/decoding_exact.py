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


def few_tolerance(o, a, q, k, scale, v_scale, n, dtype, size, softcap=0.0):
    """|error| of attention over 8-bit pages with at most 32 query rows to a KV head, whose output o (exact) alone is
    rounded (u |o|); a = Σ w|v|, size: the largest Σ|q k| scale, v_scale: the values' scales.

    Scores are sums of whole numbers, exact but for the queries': half a unit of 2^-21 of their largest value's power of
    two, so at most 2^-22 of that value.  Of an exponent in log2 units, at most E = size log2 e + |log2 of a scale| + 14,
    8 roundings of 2^-24 (three factors, two parts of the sum, the sum with log2 of the scale, that logarithm, the
    difference from the maximum); a softcap's tanh 2^-22 of the cap; the exponential 2^-23.  All of these enter a
    probability, above and below.  p · s_v is two f16 numbers, in error by 2^-22, or, below f16's normal numbers, by 2^-25
    where the largest of the wave is 2^6 or more: of n positions n 2^-31 of the largest scale times 127.  Sums of n f32
    terms, matrix sums being cut off."""
    u = torch.finfo(dtype).eps / 2
    k1 = float(k.abs().sum(-1).max()) if k.numel() else 0.0
    q1 = float(q.double().abs().max()) if q.numel() else 0.0
    s = v_scale.double().clamp(MIN)
    E = size / math.log(2) + float(s.log2().abs().max()) + 14
    p = 2.0 ** -22 * q1 * k1 * scale + math.log(2) * 8 * 2.0 ** -24 * E + softcap * 2.0 ** -21 + 2.0 ** -23
    return u * o.abs() + (2.0 ** -22 + 2 * p + 2 * (n + 16) * 2.0 ** -23) * a + n * 2.0 ** -31 * 127 * float(s.max()) + 1e-30
