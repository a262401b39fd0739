"""Rotary positions, beam selection and pools of pages on the GPU against plain forms; a search that uses them together
with the 8-bit cache."""
import math
import random

import pytest

torch = pytest.importorskip("torch")

import decoding_ref as D  # noqa: E402
import serving8_ref as R8  # noqa: E402
import serving_ref as S  # noqa: E402

pytestmark = pytest.mark.gpu
GPU = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
TYPES = [F32, F16, BF16]


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "needs the MI355X"
    from rust_interference_engine_amd import ops
    return ops


# ---- rotary positions ----

def near(out, x, positions, freqs, magnitude, interleaved):
    o, size = D.rotary(x, positions, freqs, magnitude, interleaved)
    tol = D.rotary_tolerance(o, size, magnitude, out.dtype)
    err = (out.cpu().double() - o).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("src", TYPES)
@pytest.mark.parametrize("dst", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("H,KV,hd,dims,rows", [(4, 2, 64, 64, 5), (15, 5, 64, 32, 61), (3, 1, 256, 192, 7), (2, 2, 128, 96, 2051), (5, 1, 80, 20, 9), (1, 1, 2, 2, 3), (3, 3, 33, 18, 70),
                                               (2, 1, 72, 64, 4), (2, 2, 1024, 1024, 2)])
def test_rotary(ops, H, KV, hd, dims, rows, interleaved, src, dst):
    g = torch.Generator().manual_seed(hd + dims)
    qkv = torch.randn(rows, H + 2 * KV, hd, generator=g).to(src)
    pos = torch.randint(0, 200000, (rows,), generator=g, dtype=torch.int32)
    f, _ = ops.rotary_frequencies(dims, 500000.0)
    dev = qkv.to(GPU)
    q_out, k_out = torch.empty(rows, H, hd, dtype=dst, device=GPU), torch.empty(rows, KV, hd, dtype=dst, device=GPU)
    ops.Rotary(f.to(GPU), dev[:, :H], dev[:, H:H + KV], q_out, k_out, positions=pos.to(GPU), interleaved=interleaved, magnitude=1.25)()
    near(q_out, qkv[:, :H], pos, f, 1.25, interleaved)
    near(k_out, qkv[:, H:H + KV], pos, f, 1.25, interleaved)
    assert torch.equal(dev.cpu(), qkv)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hd,dims", [(64, 64), (128, 96), (40, 18)])
def test_rotary_in_place(ops, hd, dims, interleaved, ty):
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(33, 8, hd, generator=g).to(ty)
    pos = torch.randint(0, 5000, (33,), generator=g, dtype=torch.int32)
    f, _ = ops.rotary_frequencies(dims)
    dev = qkv.to(GPU)
    ops.Rotary(f.to(GPU), dev[:, :4], dev[:, 4:6], dev[:, :4], dev[:, 4:6], positions=pos.to(GPU), interleaved=interleaved)()
    near(dev[:, :6], qkv[:, :6], pos, f, 1.0, interleaved)
    assert torch.equal(dev[:, 6:].cpu(), qkv[:, 6:])  # values are not turned
    assert torch.equal(dev[..., dims:].cpu(), qkv[..., dims:])
    q = qkv[:, :4].to(GPU)  # queries alone
    ops.Rotary(f.to(GPU), q, None, q, None, positions=pos.to(GPU), interleaved=interleaved)()
    assert torch.equal(q.cpu(), dev[:, :4].cpu())


def test_rotary_of_rows_at_any_place(ops):
    """rows that begin 2 bytes behind a boundary give the bits of aligned ones"""
    g = torch.Generator().manual_seed(2)
    flat = torch.randn(7 * 4 * 64 + 3, generator=g).to(BF16)
    pos = torch.randint(0, 5000, (7,), generator=g, dtype=torch.int32).to(GPU)
    f = ops.rotary_frequencies(48)[0].to(GPU)
    got = []
    for off in (0, 1, 3):
        buf = torch.zeros(7 * 4 * 64 + 8, dtype=BF16, device=GPU)
        x = buf[off:off + 7 * 4 * 64].view(7, 4, 64)
        x.copy_(flat[:7 * 4 * 64].view(7, 4, 64))
        out = torch.zeros_like(buf)
        o = out[off:off + 7 * 4 * 64].view(7, 4, 64)
        ops.Rotary(f, x, None, o, None, positions=pos)()
        assert bool((out[:off] == 0).all()) and bool((out[off + 7 * 4 * 64:] == 0).all())
        got.append(o.cpu())
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_of_far_and_negative_positions(ops, interleaved):
    pos = torch.tensor([0, 1, -1, 10 ** 6, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)
    x = torch.randn(7, 2, 64, generator=torch.Generator().manual_seed(3))
    f, _ = ops.rotary_frequencies(64)
    out = torch.empty(7, 2, 64, device=GPU)
    ops.Rotary(f.to(GPU), x.to(GPU), None, out, None, positions=pos.to(GPU), interleaved=interleaved)()
    o, size = D.rotary(x, pos, f, 1.0, interleaved)
    # cos and sin of 2^31 in f64 on either side: the angle's own rounding, 2^-22
    assert bool(((out.cpu().double() - o).abs() <= D.rotary_tolerance(o, size, 1.0, F32) + 2.0 ** -21 * size).all())
    assert torch.equal(out[0].cpu(), x[0])


@pytest.mark.parametrize("rows", [70, 2100])
def test_rotary_by_the_sequences_positions(ops, rows):
    lens = [(1, 1), (rows - 30, 5000), (0, 9), (5, 3), (1, 70000), (10, 10)]
    starts = torch.tensor([3] + [3 + sum(n for n, _ in lens[:i + 1]) for i in range(len(lens))], dtype=torch.int32)
    x = torch.randn(rows, 3, 64, generator=torch.Generator().manual_seed(4))
    f, _ = ops.rotary_frequencies(64)
    out = torch.full((rows, 3, 64), 7.0, device=GPU)
    seqs = ops.Seqs(starts.to(GPU), torch.tensor([n for _, n in lens], dtype=torch.int32, device=GPU), max_new=rows, max_len=70000)
    ops.Rotary(f.to(GPU), x.to(GPU), None, out, None, seqs=seqs)()
    pos = torch.cat([torch.arange(L - n, L) for n, L in lens])
    near(out[3:3 + len(pos)], x[3:3 + len(pos)], pos, f, 1.0, False)
    rest = torch.cat([out[:3], out[3 + len(pos):]])
    assert rest.numel() > 0 and bool((rest == 7.0).all())


def test_rotary_keeps_infinite_and_nan_values_to_their_pairs(ops):
    x = torch.randn(2, 1, 64, generator=torch.Generator().manual_seed(5))
    y = x.clone()
    y[0, 0, 5], y[1, 0, 40] = math.nan, math.inf
    f = ops.rotary_frequencies(64)[0].to(GPU)
    pos = torch.tensor([3, 4], dtype=torch.int32, device=GPU)
    a, b = (torch.empty(2, 1, 64, device=GPU) for _ in range(2))
    ops.Rotary(f, x.to(GPU), None, a, None, positions=pos)()
    ops.Rotary(f, y.to(GPU), None, b, None, positions=pos)()
    odd = ~torch.isfinite(b).cpu()
    assert sorted(odd.nonzero().tolist()) == [[0, 0, 5], [0, 0, 37], [1, 0, 8], [1, 0, 40]]
    assert torch.equal(a.cpu()[~odd], b.cpu()[~odd])


def test_frequencies(ops):
    f, m = ops.rotary_frequencies(8, 100.0)
    assert f.tolist() == pytest.approx([1, 100 ** -0.25, 0.1, 100 ** -0.75], rel=1e-15) and m == 1.0
    assert ops.rotary_frequencies(8, 100.0, linear=4.0)[0].tolist() == (f / 4).tolist()
    assert ops.rotary_frequencies(8, 100.0, factors=[1, 2, 4, 8])[0].tolist() == (f / torch.tensor([1.0, 2, 4, 8])).tolist()
    p, m = ops.rotary_frequencies(128, 10000.0, parts=(16.0, 4096))
    f, _ = ops.rotary_frequencies(128, 10000.0)
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(p[turns > 40], f[turns > 40]) and torch.allclose(p[turns < 0.8], f[turns < 0.8] / 16, rtol=1e-15)
    assert bool((p <= f).all()) and bool((p >= f / 16 * (1 - 1e-15)).all()) and bool((p[1:] < p[:-1]).all()) and m == pytest.approx(0.1 * math.log(16) + 1)


# ---- beam selection ----

def select(ops, logits, scores, n_out, finished=None, pad=0):
    n = scores.shape[0]
    nxt = torch.full((n, n_out), 7.0, device=GPU)
    par, tok = (torch.full((n, n_out), -7, dtype=torch.int32, device=GPU) for _ in range(2))
    call = ops.BeamSelect(logits, scores.to(GPU), nxt, par, tok, finished=None if finished is None else finished.int().to(GPU), pad=pad)
    call()
    first = nxt.cpu(), par.cpu(), tok.cpu()
    call()
    assert all(bool((a.cpu() == b).all()) for a, b in zip((nxt, par, tok), first))
    return first


def chosen(got, logits, scores, n_out, finished=None, pad=0, eps=1e-5):
    """eps: what a beam's ln of an f32 sum may be off by, tens of roundings of 2^-24"""
    n, W = scores.shape
    x = logits.cpu()
    for r in range(n):
        key, beam, token = D.beams(x[r * W:(r + 1) * W], scores[r], n_out, None if finished is None else finished[r], pad)
        nxt, par, tok = (g[r] for g in got)
        fin = key > -math.inf
        err = (nxt.double() - key).abs()[fin]
        assert bool((err <= 2.0 ** -24 * key[fin].abs() + eps).all()) and bool((nxt[~fin] == -math.inf).all())
        clear = torch.ones(n_out, dtype=torch.bool)  # neighbours in order by more than what the sums may be off, or equal beams
        gap = torch.cat([torch.full((1,), True), ((key[:-1] - key[1:]).abs() > 4 * eps) | (beam[:-1] == beam[1:]) | ~fin[1:], torch.full((1,), True)])
        clear &= gap[:-1] & gap[1:]
        clear[-1] &= False  # the next candidate may be as near
        assert bool(((par - r * W == beam) & (tok == token))[clear].all()), r
        pairs = list(zip(par.tolist(), tok.tolist()))
        assert len(set(p for p, f in zip(pairs, fin.tolist()) if f)) == int(fin.sum())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,W,V,K", [(1, 1, 1, 1), (2, 3, 2, 5), (3, 4, 7, 4), (1, 64, 100, 128), (5, 4, 1000, 8), (2, 8, 1024, 16), (2, 8, 1025, 16), (4, 5, 5003, 128), (3, 2, 32003, 4),
                                     (2, 4, 151936, 8), (1, 3, 600001, 6), (9, 1, 2049, 2)])
def test_beams(ops, n, W, V, K, dtype):
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(n * W, V, generator=g) * 3).to(dtype)
    scores = -torch.rand(n, W, generator=g) * 30
    chosen(select(ops, x.to(GPU), scores, K), x, scores, K)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_beams_of_rows_at_any_place(ops, dtype):
    g = torch.Generator().manual_seed(6)
    big = torch.randn(6, 5005, generator=g).to(dtype)
    scores = -torch.rand(2, 3, generator=g) * 3
    for off in (0, 1, 3):
        x = big.to(GPU)[:, off:off + 5001]
        chosen(select(ops, x, scores, 6), x, scores, 6)


def test_beams_that_have_ended_or_died(ops):
    g = torch.Generator().manual_seed(7)
    x = torch.randn(5 * 4, 3000, generator=g)
    scores = -torch.rand(5, 4, generator=g)
    scores[1, 1:] = -math.inf  # a search's first step
    scores[2, 0], scores[2, 2] = math.nan, math.inf
    x[3 * 4, 17], x[3 * 4 + 1, 5], x[3 * 4 + 2] = math.nan, math.inf, -math.inf
    x[4 * 4:, 3:] = -math.inf  # three tokens are allowed
    finished = torch.zeros(5, 4, dtype=torch.bool)
    finished[0, 2] = finished[1, 2] = finished[2, 3] = True
    for K in (4, 9, 20):
        chosen(select(ops, x.to(GPU), scores, K, finished, 2), x, scores, K, finished, 2)
    finished[:] = True
    got = select(ops, x.to(GPU), scores, 8, finished, 11)
    chosen(got, x, scores, 8, finished, 11)


def test_no_candidate_at_all(ops):
    x = torch.full((4, 500), -math.inf)
    got = select(ops, x.to(GPU), torch.zeros(2, 2), 3)
    assert bool((got[0] == -math.inf).all()) and got[1].tolist() == [[0, 0, 0], [2, 2, 2]] and got[2].tolist() == [[0, 1, 2]] * 2


@pytest.mark.parametrize("V", [40, 3000, 70001])
@pytest.mark.parametrize("K", [1, 5, 100])
def test_equal_beams_and_logits_go_by_number(ops, V, K):
    """every beam the same, every logit one of two values: more equals than fit a list"""
    x = torch.where(torch.arange(V) % 3 == 0, 2.0, 1.0).repeat(4, 1).to(F16)
    scores = torch.full((2, 2), -1.5)
    if K > 2 * V:  # more than there are
        from rust_interference_engine_amd import RieError
        with pytest.raises(RieError, match="n_out"):
            select(ops, x.to(GPU), scores, K)
        return
    nxt, par, tok = select(ops, x.to(GPU), scores, K)
    ids = list(range(0, V, 3)) + [i for i in range(V) if i % 3]
    want = ([(0, i) for i in ids if i % 3 == 0] + [(1, i) for i in ids if i % 3 == 0] + [(0, i) for i in ids if i % 3] + [(1, i) for i in ids if i % 3])
    # a beam's list holds its own K best: those behind come from both
    assert [list(zip(par[r].tolist(), tok[r].tolist())) for r in range(2)] == [[(2 * r + b, t) for b, t in want[:K]] for r in range(2)]
    # rows of odd length begin at other alignments; equal rows have equal sums all the same
    assert bool((nxt[0] == nxt[1]).all())


@pytest.mark.parametrize("V", [3001, 151936])
def test_few_values_above_many_equal_ones(ops, V):
    x = torch.full((2, V), -4.0)
    at = torch.randperm(V, generator=torch.Generator().manual_seed(8))[:7]
    x[0, at] = torch.arange(7).float()
    x[1, :300] = -math.inf
    scores = torch.tensor([[0.0, -0.01]])
    chosen(select(ops, x.to(GPU), scores, 20), x, scores, 20, eps=2e-5)


@pytest.mark.parametrize("mag", [1e4, 1e20, 3e38])
def test_large_logits(ops, mag):
    x = torch.randn(4, 5000, generator=torch.Generator().manual_seed(9)).clamp(-1, 1) * mag
    scores = torch.tensor([[-1.0, -2.0], [0.0, -3.0]])
    nxt, par, tok = select(ops, x.to(GPU), scores, 1)
    for r in range(2):
        assert int(par[r, 0]) == 2 * r and int(tok[r, 0]) == int(x[2 * r].argmax())
    assert bool(torch.isfinite(nxt).all())


# ---- pools of pages ----

def layouts(n_pages, page, seed):
    """caches as programs have them: a page's values in one piece, other pages' anywhere"""
    g = torch.Generator().manual_seed(seed)
    stacked = torch.randn(n_pages, 3, page, 2, 8, generator=g).half()        # layers within a page
    layered = torch.randint(-127, 128, (2, n_pages, 2, page, 32), generator=g, dtype=torch.int8)
    scales = torch.rand(2, n_pages, 1, 3, generator=g)                       # 12 bytes a page
    return stacked, layered, scales


def on_gpu(stacked, layered, scales):
    s, y, z = stacked.to(GPU), layered.to(GPU), scales.to(GPU)
    return [s[:, 0], s[:, 2], y[0], y[1].transpose(1, 2), z[0], z[1]], (s, y, z)


def cpu_of(bufs):
    return [b.cpu().contiguous() for b in bufs]


class Both:
    """A pool on the GPU beside its plain form"""

    def __init__(self, ops, rows, lens, n_pages, cols, page, seed=0, refs=None):
        self.ops = ops
        if refs is None:
            refs = [0] * n_pages
            for r in rows:
                for p in r:
                    if 0 <= p < n_pages:
                        refs[p] += 1
        self.bufs, self.keep = on_gpu(*layouts(n_pages, page, seed))
        self.ref = D.Pool(rows, lens, refs, cols, page, cpu_of(self.bufs))
        table = torch.full((len(rows), cols + 3), -1, dtype=torch.int32)
        for i, r in enumerate(rows):
            table[i, :len(r)] = torch.tensor(r, dtype=torch.int32)
        self.whole = table.to(GPU)

        def ints(x):
            return torch.tensor(x, dtype=torch.int32, device=GPU)

        self.pool = ops.PagePool(self.whole[:, :cols], ints(lens), ints([len(r) for r in rows]), ints(refs), ints([0, 0]), page_size=page)

    def check(self, caches=True):
        p, r = self.pool, self.ref
        assert p.lens.tolist() == r.lens and p.held.tolist() == [len(x) for x in r.rows]
        assert [row[:n] for row, n in zip(p.table.tolist(), p.held.tolist())] == r.rows
        assert all(x == -1 for row, n in zip(self.whole.tolist(), p.held.tolist()) for x in row[n:])
        assert p.refs.tolist() == r.refs and p.counts.tolist() == r.counts
        if caches:
            assert all(torch.equal(a, b) for a, b in zip(cpu_of(self.bufs), r.caches))
            s = self.keep[0].cpu()
            assert torch.equal(s[:, 1], layouts(s.shape[0], r.page, self.seed)[0][:, 1])  # a layer that was not named


def random_rows(rng, n, cols, page, n_pages, share=0.3):
    """rows over random pages; some begin with another row's full pages"""
    order = list(range(n_pages))
    rng.shuffle(order)
    rows, lens = [], []
    for i in range(n):
        length = rng.choice([0, 1, page, rng.randint(0, cols * page)])
        row = []
        if i and rng.random() < share:
            j = rng.randrange(i)
            row = rows[j][:min(length, lens[j]) // page]
        while len(row) < -(-length // page) and order:
            row.append(order.pop())
        if rng.random() < 0.2 and len(row) < cols and order:
            row.append(order.pop())  # reserved ahead
        length = min(length, len(row) * page)
        rows.append(row)
        lens.append(length)
    return rows, lens


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("n,cols,page,n_pages", [(1, 3, 16, 9), (4, 5, 1, 40), (12, 9, 16, 150), (70, 20, 4, 2500)])
def test_forks(ops, n, cols, page, n_pages, seed):
    rng = random.Random(seed * 100 + n)
    b = Both(ops, *random_rows(rng, n, cols, page, n_pages), n_pages, cols, page, seed)
    b.seed = seed
    src = torch.empty(n, dtype=torch.int32, device=GPU)
    fork = ops.PageFork(b.pool, src, b.bufs)
    for step in range(5):
        kind = rng.randrange(4)
        s = [rng.randrange(n) for _ in range(n)] if kind == 0 else list(range(n)) if kind == 1 else rng.sample(range(n), n) if kind == 2 else [rng.randint(-2, n + 1) for _ in range(n)]
        src.copy_(torch.tensor(s, dtype=torch.int32))
        fork()
        b.ref.fork(s)
        b.check()


def test_a_fork_that_lacks_pages(ops):
    b = Both(ops, [[3, 1], [0], [], []], [20, 5, 0, 0], 5, 4, 16)
    b.seed = 0
    src = [0, 0, 0, 1]  # two copies of a partial page, two free pages; one more of page 0
    fork = ops.PageFork(b.pool, torch.tensor(src, dtype=torch.int32, device=GPU), b.bufs)
    fork()
    b.ref.fork(src)
    b.check()
    fork()  # now three copies are wanted, and none is free
    b.ref.fork(src)
    b.check()
    assert b.pool.counts.tolist()[0] > 0


def test_a_fork_of_rows_that_are_not_in_order(ops):
    """page ids that are none, lens beyond the table, held beyond the columns"""
    b = Both(ops, [[1, -7, 2], [9999, 3], [4]], [48, 30, 16], 12, 3, 16)
    b.seed = 0
    for src in ([0, 0, 1], [1, 2, 2], [0, 0, 0]):
        ops.PageFork(b.pool, torch.tensor(src, dtype=torch.int32, device=GPU), b.bufs)()
        b.ref.fork(src)
        b.check()
    b.pool.lens.fill_(2 ** 31 - 1)
    b.pool.held.fill_(2 ** 31 - 1)
    before = b.whole[:, 3:].cpu()
    ops.PageFork(b.pool, torch.tensor([2, 0, 1], dtype=torch.int32, device=GPU), b.bufs)()
    ops.PageReserve(b.pool)()
    ops.PageCompact(b.pool, b.bufs)()
    ops.PageFree(b.pool, torch.ones(3, dtype=torch.int32, device=GPU))()
    assert torch.equal(b.whole[:, 3:].cpu(), before)  # nothing behind the columns


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("n,cols,page,n_pages", [(1, 3, 16, 9), (9, 30, 16, 200), (300, 9, 4, 3000), (1500, 4, 16, 40000)])
def test_reserve_free_and_compact(ops, n, cols, page, n_pages, seed):
    rng = random.Random(seed * 100 + n)
    b = Both(ops, *random_rows(rng, n, cols, page, n_pages), n_pages, cols, page, seed)
    b.seed = seed
    which = torch.empty(n, dtype=torch.int32, device=GPU)
    reserve, free, compact = ops.PageReserve(b.pool), ops.PageFree(b.pool, which), ops.PageCompact(b.pool, b.bufs)
    for step in range(4):
        lens = [min(x + rng.choice([0, 1, page, 3 * page]), cols * page) for x in b.ref.lens]
        b.pool.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        b.ref.lens = lens
        reserve()
        b.ref.reserve()
        b.check(False)
        gone = [int(rng.random() < 0.3) for _ in range(n)]
        which.copy_(torch.tensor(gone, dtype=torch.int32))
        free()
        b.ref.free(gone)
        b.check(False)
        if step % 2:
            compact()
            b.ref.compact()
            b.check()
            used = sum(r > 0 for r in b.ref.refs)
            assert not any(b.ref.refs[used:])


def test_a_pool_that_runs_out(ops):
    b = Both(ops, [[], [2], [], [5]], [100, 16, 40, 16], 8, 9, 16)
    b.seed = 0
    reserve = ops.PageReserve(b.pool)
    reserve()
    b.ref.reserve()
    b.check()
    assert b.pool.counts.tolist()[0] == 4
    ops.PageFree(b.pool, torch.tensor([0, 1, 0, 0], dtype=torch.int32, device=GPU))()
    b.ref.free([0, 1, 0, 0])
    reserve()
    b.ref.reserve()
    b.check()


def test_many_caches_and_pages_of_odd_sizes(ops):
    """70 buffers, more than one launch takes; pages of 4 to 20000 bytes, some unaligned"""
    n_pages, g = 11, torch.Generator().manual_seed(10)
    whole = [torch.randint(0, 255, (n_pages, 4 * (1 + 71 * i) + 4 * (i % 3)), generator=g, dtype=torch.uint8) for i in range(70)]
    dev = [w.to(GPU) for w in whole]
    view = [d[:, 4 * (i % 3):] for i, d in enumerate(dev)]
    src, dst = [3, 10, 0, -1, 4, 11], [5, 1, 7, 2, 40, 9]
    ops.PageCopy(view, torch.tensor(src, dtype=torch.int32, device=GPU), torch.tensor(dst, dtype=torch.int32, device=GPU))()
    for i, (w, d) in enumerate(zip(whole, dev)):
        w = w.clone()
        for a, b in list(zip(src, dst))[:3]:
            w[b, 4 * (i % 3):] = w[a, 4 * (i % 3):]
        assert torch.equal(d.cpu(), w), i


def test_forks_captured_and_replayed(ops):
    rng = random.Random(5)
    n, cols, page, n_pages = 8, 6, 16, 90
    b = Both(ops, *random_rows(rng, n, cols, page, n_pages), n_pages, cols, page)
    b.seed = 0
    src = torch.arange(n, dtype=torch.int32, device=GPU)
    fork, reserve = ops.PageFork(b.pool, src, b.bufs), ops.PageReserve(b.pool)
    fork(), reserve()
    b.ref.fork(list(range(n))), b.ref.reserve()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fork()
        b.pool.lens += 1
        reserve()
    for step in range(8):
        s = [rng.randrange(n) for _ in range(n)]
        src.copy_(torch.tensor(s, dtype=torch.int32))
        graph.replay()
        b.ref.fork(s)
        b.ref.lens = [x + 1 for x in b.ref.lens]
        b.ref.reserve()
        b.check()
        torch.zeros(100, device=GPU).sum().item()


# ---- together ----

def test_a_search_with_beams_over_an_8_bit_cache(ops):
    """A toy layer's search, step by step: rotary positions, append, attention, selection, fork and reserve; every step's
    attention against float64 over the codes that the beams' own histories give, every selection against the plain form."""
    torch.manual_seed(0)
    N, W, H, KV, hd, V, page, steps = 2, 3, 4, 2, 64, 300, 16, 40
    n = N * W
    g = torch.Generator().manual_seed(11)
    embed = torch.randn(V, H + 2 * KV, hd, generator=g).to(BF16)
    head = (torch.randn(H * hd, V, generator=g) * 0.15).to(GPU)
    f, m = ops.rotary_frequencies(hd, parts=(4.0, 64))
    n_pages, cols = 60, 4
    pool = ops.PagePool.empty(n_pages, n, cols, page, GPU)
    codes = torch.zeros(2, n_pages, KV, page, hd, dtype=torch.int8, device=GPU)
    scales = torch.full((2, n_pages, 1, KV), math.nan, device=GPU)
    kv = ops.PagedKv(codes[0].transpose(1, 2), codes[1].transpose(1, 2), pool.table, k_scale=scales[0], v_scale=scales[1])
    seqs = ops.Seqs(torch.arange(n + 1, dtype=torch.int32, device=GPU), pool.lens, max_new=1, max_len=cols * page)
    qkv = torch.empty(n, H + 2 * KV, hd, dtype=BF16, device=GPU)
    q, k, v = qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:]
    out, logits = torch.empty(n, H, hd, dtype=BF16, device=GPU), torch.empty(n, V, device=GPU)
    scores = torch.full((N, W), -math.inf, device=GPU)
    scores[:, 0] = 0
    nxt, parents, tokens = torch.empty(N, W, device=GPU), torch.empty(N, W, dtype=torch.int32, device=GPU), torch.empty(N, W, dtype=torch.int32, device=GPU)
    reserve, rotary = ops.PageReserve(pool), ops.Rotary(f.to(GPU), q, k, q, k, seqs=seqs, magnitude=m)
    append, attend = ops.PagedAppend(kv, seqs, k, v), ops.PagedAttention(kv, seqs, q, out)
    pick, fork = ops.BeamSelect(logits, scores, nxt, parents, tokens), ops.PageFork(pool, parents.view(-1), [codes[0], codes[1], scales[0], scales[1]])
    token = torch.arange(n) % V
    # a history's own cache: codes and scales of its blocks, as if it were alone
    alone = [[torch.zeros(cols, page, KV, hd, dtype=torch.int8) for _ in range(2)] + [torch.zeros(cols, 1, KV) for _ in range(2)] for _ in range(n)]
    for step in range(steps):
        qkv.copy_(embed[token])
        pool.lens += 1
        reserve(), rotary()
        keys, values, queries = k.float().cpu(), v.float().cpu(), q.cpu()
        near(qkv[:, :H + KV], embed[token][:, :H + KV], torch.full((n,), step), f, m, False)
        append(), attend()
        for i in range(n):
            row = torch.arange(cols)
            R8.append(alone[i][0], alone[i][2], row, page, page, step, keys[i:i + 1])
            R8.append(alone[i][1], alone[i][3], row, page, page, step, values[i:i + 1])
            x, y = ((alone[i][c].double() * alone[i][2 + c].double()[..., None]).reshape(-1, KV, hd)[:step + 1] for c in range(2))
            o, a, size = S.attend(queries[i:i + 1], x, y, step, hd ** -0.5)
            tol = R8.tolerance(o, a, queries[i:i + 1], x, y, hd ** -0.5, step + 1, hd, BF16, size)
            assert bool(((out[i:i + 1].cpu().double() - o).abs() <= tol).all()), (step, i)
        logits.copy_(out.float().view(n, -1) @ head)
        was = scores.cpu()
        pick()
        chosen((nxt.cpu(), parents.cpu(), tokens.cpu()), logits, was, W)
        fork()
        assert pool.counts.tolist()[0] == 0
        scores.copy_(nxt)
        token = tokens.view(-1).cpu().long()
        alone = [[t.clone() for t in alone[p]] for p in parents.view(-1).tolist()]
        refs = torch.bincount(pool.table[pool.table >= 0].long(), minlength=n_pages)
        assert torch.equal(refs.int(), pool.refs) and int((pool.refs > 0).sum()) <= n * (step // page + 1)
    ops.PageCompact(pool, [codes[0], codes[1], scales[0], scales[1]])()
    for i in range(n):
        t = pool.table[i, :cols][pool.table[i] >= 0].long()
        got = (codes[0][t].transpose(1, 2).double() * scales[0][t].double()[..., None]).reshape(-1, KV, hd)[:steps]
        assert torch.equal(got.cpu(), (alone[i][0].double() * alone[i][2].double()[..., None]).reshape(-1, KV, hd)[:steps])


def test_refused_on_the_gpu(ops):
    from rust_interference_engine_amd import RieError

    def refused(text, f):
        with pytest.raises(RieError, match=text):
            f()

    q = torch.randn(4, 2, 64, device=GPU)
    f = ops.rotary_frequencies(64)[0].to(GPU)
    pos = torch.zeros(4, dtype=torch.int32, device=GPU)
    refused("not both", lambda: ops.Rotary(f, q, None, q, None))
    refused("f64", lambda: ops.Rotary(f.float(), q, None, q, None, positions=pos))
    refused("positions for", lambda: ops.Rotary(f, q, None, q, None, positions=pos[:3]))
    refused("dims of heads", lambda: ops.Rotary(f, q[..., :32], None, torch.empty(4, 2, 32, device=GPU), None, positions=pos))
    refused("in place", lambda: ops.Rotary(f, q, None, q.view(2, 4, 64).transpose(0, 1), None, positions=pos)())
    refused("one GPU", lambda: ops.Rotary(f.cpu(), q, None, q, None, positions=pos))
    refused("given together", lambda: ops.Rotary(f, q, q, q, None, positions=pos))
    x, s = torch.randn(6, 100, device=GPU), torch.zeros(2, 3, device=GPU)
    o, i = torch.zeros(2, 4, device=GPU), torch.zeros(2, 4, dtype=torch.int32, device=GPU)
    refused("scores have to be", lambda: ops.BeamSelect(x[:5], s, o, i, i.clone()))
    refused("contiguous", lambda: ops.BeamSelect(x, s, o, i, i.long()))
    refused("number wanted", lambda: ops.BeamSelect(x, s, o[:1], i, i))
    refused("pad", lambda: ops.BeamSelect(x, s, o, i, i.clone(), pad=100))
    refused("n_out", lambda: ops.BeamSelect(x, s, o.repeat(1, 40), i.repeat(1, 40), i.repeat(1, 40))())
    pool = ops.PagePool.empty(9, 2, 3, 16, GPU)
    refused("one in place|columns|table", lambda: ops.PagePool(pool.table.expand(2, 3).t(), pool.lens, pool.held, pool.refs, pool.counts, page_size=16))
    refused("page_size", lambda: ops.PageReserve(ops.PagePool(pool.table, pool.lens, pool.held, pool.refs, pool.counts, page_size=24))())
    refused("a cache has to be", lambda: ops.PageCompact(pool, [torch.zeros(8, 4, device=GPU)]))
    refused("lie together", lambda: ops.PageCompact(pool, [torch.zeros(9, 4, 8, device=GPU)[:, :, :4]]))
    refused("page_bytes", lambda: ops.PageCompact(pool, [torch.zeros(9, 3, device=GPU, dtype=torch.uint8)])())
    refused("page_stride", lambda: ops.PageCompact(pool, [torch.zeros(1, 16, device=GPU).expand(9, 16)])())
    refused("src for", lambda: ops.PageFork(pool, pool.lens[:1]))
