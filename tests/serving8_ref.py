"""The paged cache in 8 bits in plain float64, and the inputs that its tests use."""
import math

import serving_ref as S
import torch

MIN, MAX = 2.0 ** -60, 2.0 ** 50


class Batch8(S.Batch):
    """A batch whose pages hold codes, and scales of blocks of `block` positions and heads [pages, blocks, heads]"""

    def __init__(self, lens, H, KV, hd, page=16, block=16, dtype=torch.float16, seed=0, **kw):
        super().__init__(lens, H, KV, hd, page=page, dtype=dtype, seed=seed, **kw)
        g = torch.Generator().manual_seed(seed + 1000)
        self.block = block
        self.k_pages, self.v_pages = (torch.randint(-127, 128, self.k_pages.shape, generator=g, dtype=torch.int8) for _ in range(2))
        self.k_scale, self.v_scale = ((torch.rand(self.n_pages, page // block, KV, generator=g) + 0.3) * 0.02 for _ in range(2))

    def values(self, codes, scale, i, upto=None):
        """[positions, KV, hd] of sequence i in float64"""
        n = self.lens[i][1] if upto is None else upto
        t = self.table[i, :-(-n // self.page)].long()
        x = self.paged(codes)[t].double() * scale[t].double().repeat_interleave(self.block, 1)[..., None]
        return x.reshape(-1, self.KV, self.hd)[:n]


def tolerance(o, a, q, k, v, scale, n, hd, dtype, size, softcap=0.0):
    """|error| of the kernels' output o (exact), a = Σ w|v|, q, k, v as they are read; size: the largest Σ|q k| scale.

    The output is rounded once (u |o|).  A probability times its value's scale is an f16 number, in error by half a step
    (2^-11), or, below f16's normal numbers, by 2^-25 where the largest is at least 2^-2 (so of n positions at most n 2^-23
    times the largest |v|).  Scores: f32 sums of hd products of f16 numbers and codes (hd + 4 roundings of 2^-23, matrix
    sums being cut off), or whole numbers of 2^-23 of a query's largest value; the factors' and the exponent's roundings, 8
    of 2^-24 of exponents of at most (score + 64) / ln 2, in log2 units, 64 being more than log2 of a scale; a softcap's tanh
    2^-22 of the cap.  All of these enter a probability, above and below.  Sums of n f32 terms."""
    u = torch.finfo(dtype).eps / 2
    k1 = float(k.abs().sum(-1).max()) if k.numel() else 0.0
    q1 = float(q.double().abs().max()) if q.numel() else 0.0
    score = (hd + 4) * 2.0 ** -23 * size + 2.0 ** -23 * q1 * k1 * scale + 2.0 ** -21 * (size + 64) + softcap * 2.0 ** -21
    most = float(v.abs().max()) if v.numel() else 0.0
    return u * o.abs() + (2.0 ** -11 + 2 * score + 2 * (n + 16) * 2.0 ** -23) * a + n * 2.0 ** -23 * most + 1e-30


def append(codes, scale, table, page, block, first, x):
    """x [new, KV, hd] to positions first.. of a sequence; codes [pages, page, KV, hd] and scale [pages, blocks, KV] in place"""
    x = x.double()
    n, L = x.shape[0], first + x.shape[0]
    p = first
    while p < L:
        b0 = p // block * block
        e = min(b0 + block, L)
        pg, slot, nb = int(table[p // page]), b0 % page, b0 % page // block
        y = x[p - first:e - first]
        if 0 <= pg < codes.shape[0]:
            for h in range(x.shape[1]):
                was = float(scale[pg, nb, h]) if p > b0 else 0.0
                most = y[:, h].abs().max()
                now = float((most / 127).float())
                now = 0.0 if now < MIN else now
                if not bool(torch.isfinite(y[:, h]).all()) or now > MAX or not 0 <= was <= MAX:
                    now = math.nan
                else:
                    now = max(now, was)
                scale[pg, nb, h] = now
                if now > was and p > b0:
                    old = codes[pg, slot:slot + p - b0, h]
                    codes[pg, slot:slot + p - b0, h] = (old.double() * (was / now)).round().to(torch.int8)
                at = slice(slot + p - b0, slot + e - b0)
                codes[pg, at, h] = (y[:, h] * (1 / now)).round().to(torch.int8) if now > 0 else 0
        p = e
    return n
