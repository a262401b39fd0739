"""Plain float64 forms of the batched serving operators, and the inputs that their tests use."""
import math

import torch


def attend(q, k, v, pos0, scale, window=0, softcap=0.0):
    """q [new, H, hd], k and v [len, KV, hd] of one sequence, token t at position pos0 + t: outputs,
    Σ w|v| and Σ|q k| scale, the last two for the error bound"""
    q, k, v = q.double(), k.double(), v.double()
    H, KV = q.shape[1], k.shape[1]
    n, L = q.shape[0], k.shape[0]
    k, v = (x.repeat_interleave(H // KV, 1).transpose(0, 1) for x in (k, v))  # [H, L, hd]
    q = q.transpose(0, 1)
    s = (q @ k.transpose(1, 2)) * scale
    size = (q.abs() @ k.abs().transpose(1, 2)) * scale
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    p = pos0 + torch.arange(n)[:, None]
    j = torch.arange(L)[None]
    seen = j <= p
    if window:
        seen &= j > p - window
    s = s.masked_fill(~seen, -math.inf)
    m = s.amax(-1, keepdim=True) if L else torch.full((H, n, 1), -math.inf, dtype=torch.float64)
    e = torch.where(seen, torch.exp(s - m.masked_fill(m == -math.inf, 0.0)), 0.0)
    w = e / e.sum(-1, keepdim=True).clamp(min=1e-300)
    vz = torch.where(seen.any(0)[:, None], v, 0.0)  # values that nobody sees
    o = w @ vz
    return o.transpose(0, 1), (w @ vz.abs()).transpose(0, 1), float(size.masked_fill(~seen, 0.0).max()) if L and n else 0.0


def tolerance(o, a, size, n, hd, dtype, softcap=0.0):
    """|error| of the kernel's output o (exact), a = Σ w|v|.  u = half a step of the type: the output is rounded once
    (u|o|); each probability once, in the numerator and in the sum that divides it (2 u a together).  Scores are f32
    sums of hd products (hd + 4 roundings of at most 2^-23 of Σ|q k|, matrix sums being cut off), the softcap's tanh is
    off by 2^-22 of the cap; either enters the numerator's and the sum's exponentials.  Sums of n f32 terms."""
    u = torch.finfo(dtype).eps / 2
    score = (hd + 4) * 2.0 ** -23 * size + softcap * 2.0 ** -21
    return u * o.abs() + (2 * u + 2 * score + 2 * (n + 16) * 2.0 ** -23) * a + 1e-30


def logprobs(x, targets, top):
    x = x.double()
    p = torch.log_softmax(x, -1)
    h = -torch.where(p == -math.inf, 0.0, p.exp() * p).sum(-1)
    t = targets.long()
    ok = (t >= 0) & (t < x.shape[1])
    lp = torch.where(ok, p.gather(1, t.clamp(0, x.shape[1] - 1)[:, None])[:, 0], math.nan)
    rank = torch.where(x.isnan(), -math.inf, x) + 0.0
    ids = rank.sort(dim=-1, descending=True, stable=True).indices[:, :top]
    return lp, h, ids, p.gather(1, ids)


class Batch:
    """Sequences of (new tokens, positions with them) over shuffled pages, on the CPU; rows behind the last one's too."""

    def __init__(self, lens, H, KV, hd, page=16, dtype=torch.float16, seed=0, extra_rows=0, extra_cols=0, order="heads"):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.H, self.KV, self.hd, self.page, self.dtype = lens, H, KV, hd, page, dtype
        starts = [0]
        for n, _ in lens:
            starts.append(starts[-1] + n)
        self.starts = torch.tensor(starts, dtype=torch.int32)
        self.L = torch.tensor([x for _, x in lens], dtype=torch.int32)
        self.rows = starts[-1] + extra_rows
        need = [-(-x // page) for _, x in lens]
        self.n_pages = sum(need) + 2
        order_ = torch.randperm(self.n_pages, generator=g).int()
        self.table = torch.full((len(lens), max(1, max(need)) + extra_cols), self.n_pages + 7, dtype=torch.int32)  # none of the pages
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order_[at:at + n]
            at += n
        shape = (self.n_pages, KV, page, hd) if order == "heads" else (self.n_pages, page, KV, hd)
        mk = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.k_pages, self.v_pages = mk(*shape).to(dtype), mk(*shape).to(dtype)
        self.order = order
        self.q = (mk(max(self.rows, 1), H, hd) * 1.3).to(dtype)

    def paged(self, pages):
        return pages.transpose(1, 2) if self.order == "heads" else pages

    def cached(self, pages, i, upto=None):
        """[positions, KV, hd] of sequence i"""
        n = self.lens[i][1] if upto is None else upto
        t = self.table[i, :-(-n // self.page)].long()
        return self.paged(pages)[t].reshape(-1, self.KV, self.hd)[:n]

    def max_new(self):
        return max(1, max(n for n, _ in self.lens))

    def max_len(self):
        return max(1, max(x for _, x in self.lens))
