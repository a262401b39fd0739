"""Plain forms of rotary positions, beam selection and the pool of pages, for their tests."""
import math

import torch


def rotary(x, positions, freqs, magnitude, interleaved):
    """x [rows, heads, size] turned, in float64, and the sizes |x| + |y| of every pair for the error bound"""
    x = x.double()
    d = 2 * freqs.numel()
    a = positions.double()[:, None] * freqs.double()
    c, s = (magnitude * f(a)[:, None] for f in (torch.cos, torch.sin))
    u, v = (x[..., 0:d:2], x[..., 1:d:2]) if interleaved else (x[..., :d // 2], x[..., d // 2:d])

    def joined(p, q, rest):
        y = torch.stack([p, q], -1).flatten(-2) if interleaved else torch.cat([p, q], -1)
        return torch.cat([y, rest], -1)

    size = u.abs() + v.abs()
    return joined(u * c - v * s, u * s + v * c, x[..., d:]), joined(size, size, 0 * x[..., d:])


def rotary_tolerance(o, size, magnitude, dtype):
    """The output is rounded once; sine and cosine are off by 2^-23 (two units) and by 2^-25 of the angle's rounding within
    an eighth of a turn, their product with the magnitude, both products and the sum by 2^-24 each: under 2^-21 of |x| + |y|."""
    u = torch.finfo(dtype).eps / 2
    return u * o.abs() + 2.0 ** -21 * abs(magnitude) * size + torch.finfo(dtype).tiny * u * 2


def beams(logits, scores, n_out, finished=None, pad=0):
    """of one request [beams, vocabulary]: sums of the best in order, beams, tokens, in float64"""
    W, V = logits.shape
    x = logits.double()
    key = scores.double()[:, None] + torch.log_softmax(x, -1)
    dead = ~torch.isfinite(scores) | x.isnan().any(-1) | (x == math.inf).any(-1) | (x == -math.inf).all(-1)
    key[dead] = -math.inf
    out = []
    for b in range(W):
        if finished is not None and bool(finished[b]):
            own = float(scores[b]) if bool(torch.isfinite(scores[b])) else -math.inf
            out += [(-own if i == 0 else math.inf, b, i, pad) for i in range(min(n_out, V))]
            continue
        rank = torch.zeros(V, dtype=torch.float64) if bool(dead[b]) else x[b]
        ids = (rank + 0.0).sort(descending=True, stable=True).indices[:n_out].tolist()
        out += [(-float(key[b, t]), b, i, t) for i, t in enumerate(ids)]
    out.sort(key=lambda c: c[:3])
    out = out[:n_out]
    return torch.tensor([-c[0] for c in out], dtype=torch.float64), torch.tensor([c[1] for c in out]), torch.tensor([c[3] for c in out])


class Pool:
    """The pool in plain Python: rows of pages, positions, references, and the caches' pages"""

    def __init__(self, rows, lens, refs, cols, page, caches=()):
        self.rows, self.lens, self.refs, self.cols, self.page = [list(r) for r in rows], list(lens), list(refs), cols, page
        self.caches = [c.clone() for c in caches]
        self.counts = [0, 0]

    def free_pages(self):
        return [p for p, r in enumerate(self.refs) if r == 0]

    def known(self, p):
        return 0 <= p < len(self.refs)

    def size(self, i):
        n = min(max(self.lens[i], 0), self.cols * self.page)
        return n // self.page, -(-n // self.page)

    def reserve(self):
        free, lacked = self.free_pages(), 0
        for i, r in enumerate(self.rows):
            for _ in range(max(0, self.size(i)[1] - len(r))):
                if free:
                    p = free.pop(0)
                    r.append(p)
                    self.refs[p] = 1
                else:
                    lacked += 1
        self.counts[0] = lacked

    def fork(self, src):
        n, free = len(self.rows), self.free_pages()
        heir, rows, lens, copies, lacked = {}, [], [], [], 0
        for i, r in enumerate(src):
            if 0 <= r < n and (r == i or r not in heir):
                heir[r] = i if r == i or src[r] != r else r
        for i, r in enumerate(src):
            if not 0 <= r < n:
                rows.append([])
                lens.append(0)
                continue
            full, touched = self.size(r)
            old = self.rows[r]
            lens.append(self.lens[r])
            if heir[r] == i:
                rows.append(list(old))
                continue
            row = old[:touched]
            if touched > full and len(old) > full:
                if free:
                    p = free.pop(0)
                    if self.known(old[full]):
                        copies.append((old[full], p))
                    row[full] = p
                else:
                    row[full] = -1
                    lacked += 1
            rows.append(row)
        for r in self.rows:
            for p in r:
                if self.known(p):
                    self.refs[p] -= 1
        for row in rows:
            for p in row:
                if self.known(p):
                    self.refs[p] += 1
        for c in self.caches:
            for a, b in copies:
                c[b] = c[a]
        self.rows, self.lens, self.counts[0] = rows, lens, lacked

    def free(self, which):
        for i, w in enumerate(which):
            if w:
                for p in self.rows[i]:
                    if self.known(p):
                        self.refs[p] -= 1
                self.rows[i], self.lens[i] = [], 0

    def compact(self):
        used = sum(r > 0 for r in self.refs)
        a, b = [p for p, r in enumerate(self.refs) if r > 0 and p >= used], [p for p in self.free_pages() if p < used]
        goes = dict(zip(a, b))
        for x, y in goes.items():
            self.refs[y], self.refs[x] = self.refs[x], 0
            for c in self.caches:
                c[y] = c[x]
        self.rows = [[goes.get(p, p) for p in r] for r in self.rows]
        self.counts[1] = used
