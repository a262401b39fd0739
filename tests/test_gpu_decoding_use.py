"""The 8-bit cache's tile attention where a launch is divided into pieces, and rotary positions, beam selection and pools
as a program uses them: captured and replayed over new contents, on two streams at once, with rows that bring nothing."""
import math
import random

import pytest

torch = pytest.importorskip("torch")

import serving8_ref as R  # noqa: E402
import serving_ref as S  # noqa: E402
from test_gpu_decoding import Both, chosen, near, random_rows  # noqa: E402
from test_gpu_serving8 import check, paged  # noqa: E402

pytestmark = pytest.mark.gpu
GPU = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "needs the MI355X"
    from rust_interference_engine_amd import ops
    return ops


def settle():
    """the program's own work between replays"""
    torch.zeros(1000, device=GPU).sum().item()
    torch.cuda.synchronize()


# ---- tiles in pieces ----

@pytest.mark.parametrize("H,KV,hd,page,dtype", [(4, 1, 32, 16, F16), (8, 2, 64, 64, BF16), (6, 3, 96, 32, F16), (8, 2, 128, 128, BF16), (7, 7, 128, 16, F16), (4, 1, 256, 32, BF16)])
@pytest.mark.parametrize("window,softcap", [(0, 0.0), (900, 0.0), (0, 3.0), (1300, 2.0)])
def test_sequences_that_several_workgroups_share(ops, H, KV, hd, page, dtype, window, softcap):
    b = R.Batch8([(1, 9), (200, 2900), (0, 50), (33, 33), (90, 5000), (1, 1), (300, 300), (17, 1700)], H, KV, hd, page=page, dtype=dtype, seed=31, extra_rows=5)
    check(b, paged(ops, b, window, softcap), window, softcap)


@pytest.mark.parametrize("n_seq,hd", [(300, 64), (1500, 32), (70, 128)])
def test_many_sequences_with_loose_bounds(ops, n_seq, hd):
    """short sequences under bounds that would hold far longer ones, and one long one among them"""
    rng = random.Random(n_seq)
    lens = [(n, n + rng.choice([0, 1, 60, 200])) for n in (rng.choice([0, 1, 1, 2, 40]) for _ in range(n_seq))]
    lens[n_seq // 2] = (130, 4500)
    b = R.Batch8(lens, 4, 2, hd, page=32, block=32, dtype=F16, seed=32)
    check(b, paged(ops, b, max_new=5000, max_len=9000))


def test_a_nan_scale_in_one_of_the_pieces(ops):
    b = R.Batch8([(150, 4000), (70, 3000)], 8, 2, 64, page=64, block=64, dtype=F16, seed=33)
    b.k_scale[b.table[0, 20], 0, 1] = math.nan  # position 1280 on, of head 1, of the first sequence
    out = paged(ops, b)
    bad = out[:150, 4:]
    assert bool(bad.isnan().all())
    keep = b.k_scale.clone()
    b.k_scale[b.table[0, 20], 0, 1] = 0.01
    whole = paged(ops, b)
    assert torch.equal(out[:150, :4], whole[:150, :4]) and torch.equal(out[150:], whole[150:])
    b.k_scale = keep
    out = paged(ops, b, window=1000)  # only tokens from before position 2344 see it, and there are none
    assert not bool(out.isnan().any())


def test_chunks_captured_and_replayed_over_other_lengths(ops):
    b = R.Batch8([(60, 2000), (40, 2000), (100, 2000)], 8, 2, 64, page=64, block=64, dtype=F16, seed=34)
    kv = ops.PagedKv(b.paged(b.k_pages.to(GPU)), b.paged(b.v_pages.to(GPU)), b.table.to(GPU), k_scale=b.k_scale.to(GPU), v_scale=b.v_scale.to(GPU))
    starts, lens, q = b.starts.to(GPU), b.L.to(GPU), b.q.to(GPU)
    out = torch.empty_like(q)
    call = ops.PagedAttention(kv, ops.Seqs(starts, lens, max_new=200, max_len=2000), q, out)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for new, length in (((60, 40, 100), (2000, 2000, 2000)), ((1, 198, 1), (60, 1999, 1)), ((0, 0, 200), (0, 500, 300)), ((200, 0, 0), (1234, 0, 9)), ((60, 40, 100), (100, 1500, 700))):
        b.lens = list(zip(new, length))
        ends = torch.tensor([0, new[0], new[0] + new[1], sum(new)], dtype=torch.int32)
        b.starts = ends
        starts.copy_(ends)
        lens.copy_(torch.tensor(length, dtype=torch.int32))
        out.fill_(7.0)
        graph.replay()
        check(b, out.cpu())
        settle()


def test_two_chunks_at_once_on_two_streams(ops):
    b = R.Batch8([(80, 5000), (64, 64), (30, 2500)], 8, 2, 128, page=64, block=32, dtype=BF16, seed=35)
    kv = ops.PagedKv(b.paged(b.k_pages.to(GPU)), b.paged(b.v_pages.to(GPU)), b.table.to(GPU), k_scale=b.k_scale.to(GPU), v_scale=b.v_scale.to(GPU))
    seqs = ops.Seqs(b.starts.to(GPU), b.L.to(GPU), max_new=80, max_len=5000)
    q = [b.q.to(GPU), -b.q.to(GPU)]
    out = [torch.empty_like(x) for x in q]
    calls = [ops.PagedAttention(kv, seqs, x, o) for x, o in zip(q, out)]
    for c in calls:
        c()
    want = [o.cpu() for o in out]
    streams = [torch.cuda.Stream() for _ in q]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, s in zip(calls, streams):
            c(stream=s)
    torch.cuda.synchronize()
    assert all(torch.equal(o.cpu(), w) for o, w in zip(out, want))


@pytest.mark.parametrize("max_new", [1, 60])
def test_a_batch_that_brings_nothing(ops, max_new):
    """rows behind the last sequence only: neither the outputs nor the cache change"""
    b = R.Batch8([(0, 40), (0, 0), (0, 3000)], 8, 2, 64, page=32, dtype=F16, seed=36, extra_rows=70)
    out = paged(ops, b, max_new=max_new, max_len=3000)
    assert bool((out == 7.0).all())
    dev = [x.to(GPU) for x in (b.k_pages, b.v_pages, b.k_scale, b.v_scale)]
    kv = ops.PagedKv(b.paged(dev[0]), b.paged(dev[1]), b.table.to(GPU), k_scale=dev[2], v_scale=dev[3])
    x = torch.randn(b.rows, 2, 64, device=GPU)
    ops.PagedAppend(kv, ops.Seqs(b.starts.to(GPU), b.L.to(GPU), max_new=max_new, max_len=3000), x, x.clone())()
    assert all(torch.equal(d.cpu(), h) for d, h in zip(dev, (b.k_pages, b.v_pages, b.k_scale, b.v_scale)))


# ---- rotary positions ----

@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_captured_and_replayed_as_sequences_move_on(ops, interleaved):
    g = torch.Generator().manual_seed(41)
    f = ops.rotary_frequencies(64)[0]
    starts, lens = torch.tensor([0, 3, 3, 10], dtype=torch.int32), torch.tensor([5, 90, 7], dtype=torch.int32)
    d_starts, d_lens = starts.to(GPU), lens.to(GPU)
    q, k = torch.empty(12, 6, 64, dtype=BF16, device=GPU), torch.empty(12, 2, 64, dtype=BF16, device=GPU)
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    call = ops.Rotary(f.to(GPU), q, k, q_out, k_out, seqs=ops.Seqs(d_starts, d_lens, max_new=12, max_len=100000), interleaved=interleaved)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for step, cuts in enumerate(((0, 3, 3, 10), (0, 0, 12, 12), (0, 1, 2, 3), (0, 12, 12, 12))):
        hq, hk = torch.randn(12, 6, 64, generator=g).to(BF16), torch.randn(12, 2, 64, generator=g).to(BF16)
        L = torch.tensor([12 + 1000 * step, 30 + step, 99999 - step], dtype=torch.int32)
        q.copy_(hq), k.copy_(hk), d_lens.copy_(L), d_starts.copy_(torch.tensor(cuts, dtype=torch.int32))
        q_out.fill_(7.0), k_out.fill_(7.0)
        graph.replay()
        pos = torch.cat([torch.arange(int(L[i]) - (b - a), int(L[i])) for i, (a, b) in enumerate(zip(cuts, cuts[1:]))])
        n = cuts[-1]
        for out, x in ((q_out, hq), (k_out, hk)):
            near(out[:n], x[:n], pos, f, 1.0, interleaved)
            assert bool((out[n:] == 7.0).all())
        settle()


def test_rotary_of_queries_in_place_and_keys_to_another_place(ops):
    """heads of a fused projection; the values behind the rotated ones are copied only where the output lies elsewhere"""
    g = torch.Generator().manual_seed(42)
    f = ops.rotary_frequencies(32)[0]
    h = torch.randn(40, 9, 64, generator=g).half()
    pos = torch.randint(0, 5000, (40,), generator=g).int()
    x = h.to(GPU)
    k_out = torch.empty(40, 2, 64, dtype=F16, device=GPU)
    ops.Rotary(f.to(GPU), x[:, :5], x[:, 5:7], x[:, :5], k_out, positions=pos.to(GPU))()
    near(x[:, :5], h[:, :5], pos, f, 1.0, False)
    near(k_out, h[:, 5:7], pos, f, 1.0, False)
    assert torch.equal(x[:, 5:].cpu(), h[:, 5:]) and torch.equal(x[:, :5, 32:].cpu(), h[:, :5, 32:]) and torch.equal(k_out[..., 32:].cpu(), h[:, 5:7, 32:])


# ---- beam selection ----

def test_beams_captured_and_replayed(ops):
    """3 requests of 5 beams: every replay over new logits, sums and ends; workspaces keep nothing"""
    g = torch.Generator().manual_seed(43)
    x, scores, finished = torch.empty(15, 20011, dtype=BF16, device=GPU), torch.zeros(3, 5, device=GPU), torch.zeros(3, 5, dtype=torch.int32, device=GPU)
    x.zero_()
    nxt = torch.empty(3, 10, device=GPU)
    par, tok = (torch.empty(3, 10, dtype=torch.int32, device=GPU) for _ in range(2))
    call = ops.BeamSelect(x, scores, nxt, par, tok, finished=finished, pad=3)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for step in range(6):
        h, s, f = (torch.randn(15, 20011, generator=g) * 3).to(BF16), -torch.rand(3, 5, generator=g) * 9, torch.rand(3, 5, generator=g) < 0.1 * step
        x.copy_(h), scores.copy_(s), finished.copy_(f)
        graph.replay()
        chosen((nxt.cpu(), par.cpu(), tok.cpu()), h, s, 10, f, 3)
        settle()


def test_two_selections_at_once_on_two_streams(ops):
    g = torch.Generator().manual_seed(44)
    x = [(torch.randn(32, 50000, generator=g) * 2).to(GPU) for _ in range(2)]
    s = [-torch.rand(4, 8, generator=g).to(GPU) for _ in range(2)]
    out = [(torch.empty(4, 16, device=GPU), torch.empty(4, 16, dtype=torch.int32, device=GPU), torch.empty(4, 16, dtype=torch.int32, device=GPU)) for _ in range(2)]
    calls = [ops.BeamSelect(a, b, *o) for a, b, o in zip(x, s, out)]
    for c in calls:
        c()
    want = [[t.cpu() for t in o] for o in out]
    streams = [torch.cuda.Stream() for _ in x]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, st in zip(calls, streams):
            c(stream=st)
    torch.cuda.synchronize()
    assert all(torch.equal(t.cpu(), w) for o, ws in zip(out, want) for t, w in zip(o, ws))


def test_one_row_of_logits_for_all_beams(ops):
    """the first step of a search: logits of one row, expanded over the beams, of which one counts"""
    g = torch.Generator().manual_seed(45)
    x = torch.randn(1, 9001, generator=g)
    scores = torch.full((1, 6), -math.inf)
    scores[0, 0] = 0
    nxt, par, tok = torch.empty(1, 6, device=GPU), *(torch.empty(1, 6, dtype=torch.int32, device=GPU) for _ in range(2))
    ops.BeamSelect(x.to(GPU).expand(6, 9001), scores.to(GPU), nxt, par, tok)()
    chosen((nxt.cpu(), par.cpu(), tok.cpu()), x.expand(6, 9001), scores, 6)
    assert not bool(par.any()) and tok[0].tolist() == x[0].topk(6).indices.tolist()


# ---- pools ----

def test_reserve_free_and_compact_captured_and_replayed(ops):
    rng = random.Random(46)
    n, cols, page, n_pages = 20, 12, 16, 260
    b = Both(ops, *random_rows(rng, n, cols, page, n_pages), n_pages, cols, page)
    b.seed = 0
    which = torch.zeros(n, dtype=torch.int32, device=GPU)
    reserve, free, compact = ops.PageReserve(b.pool), ops.PageFree(b.pool, which), ops.PageCompact(b.pool, b.bufs)
    reserve(), free(), compact()
    b.ref.reserve(), b.ref.free([0] * n), b.ref.compact()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        reserve(), free(), compact()
    for step in range(6):
        lens = [min(x + rng.choice([0, 1, page, 3 * page]), cols * page) for x in b.ref.lens]
        gone = [int(rng.random() < 0.3) for _ in range(n)]
        b.pool.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        which.copy_(torch.tensor(gone, dtype=torch.int32))
        b.ref.lens = lens
        graph.replay()
        b.ref.reserve(), b.ref.free(gone), b.ref.compact()
        b.check()
        settle()


def test_the_largest_number_of_sequences(ops):
    """4096 rows, of which every one takes another's place, and a pool of more pages than one round of the search"""
    rng = random.Random(47)
    n, cols, page, n_pages = 4096, 5, 4, 70000
    b = Both(ops, *random_rows(rng, n, cols, page, n_pages), n_pages, cols, page)
    b.seed = 0
    src = [rng.randrange(n) for _ in range(n)]
    src[5], src[6], src[4095] = -1, n, 2 ** 31 - 1
    ops.PageFork(b.pool, torch.tensor(src, dtype=torch.int32, device=GPU), b.bufs)()
    b.ref.fork(src)
    b.check()
    lens = [min(x + rng.randrange(9), cols * page) for x in b.ref.lens]
    b.pool.lens.copy_(torch.tensor(lens, dtype=torch.int32))
    b.ref.lens = lens
    ops.PageReserve(b.pool)()
    b.ref.reserve()
    ops.PageCompact(b.pool, b.bufs)()
    b.ref.compact()
    b.check()


def test_numbers_that_are_none_stay_in_bounds(ops):
    """a pool whose memory holds anything: every call ends and touches nothing outside it"""
    g = torch.Generator().manual_seed(48)
    guard = torch.full((3, 40, 64), 9, dtype=torch.uint8, device=GPU)
    for seed in range(20):
        wild = [2 ** 31 - 1, -2 ** 31, -1, 0, 1, 39, 40, 41, 77]

        def some(*shape):
            return torch.tensor(wild, dtype=torch.int32)[torch.randint(0, len(wild), shape, generator=g)].to(GPU)

        whole = torch.full((8, 9), -5, dtype=torch.int32, device=GPU)
        whole[1:7, :6] = some(6, 6)
        before = whole.clone()
        pool = ops.PagePool(whole[1:7, :6], some(6), some(6), some(40), some(2), page_size=16)
        cache = guard[1]
        for call in (ops.PageReserve(pool), ops.PageFork(pool, some(6), [cache]), ops.PageFree(pool, some(6)), ops.PageCompact(pool, [cache]), ops.PageCopy([cache], some(9), some(9))):
            call()
        torch.cuda.synchronize()
        assert torch.equal(whole[0], before[0]) and torch.equal(whole[7], before[7]) and torch.equal(whole[:, 6:], before[:, 6:])
        assert bool((guard == 9).all())


# ---- single tokens in pieces ----

@pytest.mark.parametrize("H,KV,hd,page,dtype", [(4, 1, 32, 16, F16), (8, 2, 64, 64, BF16), (6, 3, 96, 32, F16), (8, 2, 128, 128, BF16), (32, 1, 128, 16, F16), (4, 1, 256, 32, BF16), (9, 9, 64, 16, F16)])
@pytest.mark.parametrize("window,softcap", [(0, 0.0), (700, 0.0), (0, 3.0)])
def test_few_rows_that_several_workgroups_share(ops, H, KV, hd, page, dtype, window, softcap):
    G = H // KV
    some = max(1, 32 // G)
    b = R.Batch8([(1, 9), (some, 2900), (0, 50), (1, 5000), (1, 1), (some, some), (1, 1700), (1, 0), (1, 128), (1, 129)], H, KV, hd, page=page, dtype=dtype, seed=51, extra_rows=5)
    check(b, paged(ops, b, window, softcap), window, softcap)


@pytest.mark.parametrize("n_seq", [2, 64, 65, 200, 700])
def test_pieces_of_many_sequences(ops, n_seq):
    """more sequences than a wave scans at once; lengths from none to many pieces, under a loose bound"""
    rng = random.Random(n_seq)
    lens = [(rng.choice([0, 1, 1, 2]), rng.choice([0, 1, 60, 127, 128, 300, 900])) for _ in range(n_seq)]
    lens = [(min(n, x), x) for n, x in lens]
    lens[-1], lens[n_seq // 2] = (1, 6000), (2, 3500)
    b = R.Batch8(lens, 4, 2, 64, page=32, block=32, dtype=F16, seed=52)
    check(b, paged(ops, b, max_len=20000))
    check(b, paged(ops, b, window=200, max_len=20000), window=200)


def test_lengths_beyond_the_bound_stay_in_bounds(ops):
    """lengths that pass max_len, up to all that a table addresses, over pages used again and again: every call ends, what it
    should not write stays, and a sequence that passes the bound is whole all the same"""
    n_pages, KV, hd, page, cols = 9, 2, 64, 4096, 2000
    codes = torch.randint(-127, 128, (2, n_pages, KV, page, hd), dtype=torch.int8, generator=torch.Generator().manual_seed(53))
    scale = torch.full((2, n_pages, 1, KV), 0.01)
    table = (torch.arange(40 * cols, dtype=torch.int32) % n_pages).view(40, cols)
    dev, s = codes.to(GPU), scale.to(GPU)
    kv = ops.PagedKv(*dev.transpose(2, 3), table.to(GPU), k_scale=s[0], v_scale=s[1])
    starts = torch.arange(41, dtype=torch.int32, device=GPU)
    lens = torch.full((40,), 1000, dtype=torch.int32, device=GPU)
    lens[3], lens[7], lens[20] = 2 ** 31 - 1, 30000, -5
    out = torch.full((44, 4, hd), 7.0, dtype=F16, device=GPU)
    q = (torch.randn(44, 4, hd, generator=torch.Generator().manual_seed(54)) * 8).half()  # few positions count, so that a missing part shows
    ops.PagedAttention(kv, ops.Seqs(starts, lens, max_new=1, max_len=1000), q.to(GPU), out)()
    torch.cuda.synchronize()
    assert bool((out[40:] == 7.0).all()) and bool(out[:40].isfinite().all()) and bool((out[20] == 0).all())
    k, v = ((codes[i][table[7, :8].long()].double() * scale[i, 0, 0, 0].double()).transpose(1, 2).reshape(-1, KV, hd)[:30000] for i in range(2))
    o, a, size = S.attend(q[7:8], k, v, 29999, hd ** -0.5)
    tol = R.tolerance(o, a, q[7:8], k, v, hd ** -0.5, 30000, hd, F16, size)
    assert bool(((out[7:8].cpu().double() - o).abs() <= tol).all())


def test_single_tokens_captured_and_replayed_over_other_lengths(ops):
    """the cuts move with the lengths; two graphs with a workspace each, replayed in turn"""
    b = R.Batch8([(1, 4000)] * 5, 8, 2, 64, page=64, block=64, dtype=F16, seed=55)
    kv = ops.PagedKv(b.paged(b.k_pages.to(GPU)), b.paged(b.v_pages.to(GPU)), b.table.to(GPU), k_scale=b.k_scale.to(GPU), v_scale=b.v_scale.to(GPU))
    starts, lens, q = b.starts.to(GPU), b.L.to(GPU), b.q.to(GPU)
    out = [torch.empty_like(q) for _ in range(2)]
    calls = [ops.PagedAttention(kv, ops.Seqs(starts, lens, max_new=3, max_len=4000), q, o) for o in out]
    graphs = []
    for call in calls:
        call()
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            call()
    for new, length in (((1, 1, 1, 1, 1), (4000, 1, 128, 129, 0)), ((0, 3, 0, 2, 0), (9, 4000, 0, 3999, 4000)), ((0, 0, 0, 0, 1), (0, 0, 0, 0, 4000)), ((1, 1, 1, 1, 1), (1, 1, 1, 1, 1)), ((1, 1, 1, 1, 1), (4000,) * 5)):
        b.lens = list(zip(new, length))
        b.starts = torch.tensor([sum(new[:i]) for i in range(6)], dtype=torch.int32)
        starts.copy_(b.starts)
        lens.copy_(torch.tensor(length, dtype=torch.int32))
        for graph, o in zip(graphs, out):
            o.fill_(7.0)
            graph.replay()
        for o in out:
            check(b, o.cpu())
        settle()


def test_two_batches_of_single_tokens_at_once_on_two_streams(ops):
    b = R.Batch8([(1, 5000), (1, 100), (1, 3000), (1, 1)], 8, 2, 128, page=64, block=32, dtype=BF16, seed=56)
    kv = ops.PagedKv(b.paged(b.k_pages.to(GPU)), b.paged(b.v_pages.to(GPU)), b.table.to(GPU), k_scale=b.k_scale.to(GPU), v_scale=b.v_scale.to(GPU))
    seqs = ops.Seqs(b.starts.to(GPU), b.L.to(GPU), max_new=1, max_len=5000)
    q = [b.q.to(GPU), -b.q.to(GPU)]
    out = [torch.empty_like(x) for x in q]
    calls = [ops.PagedAttention(kv, seqs, x, o) for x, o in zip(q, out)]
    for c in calls:
        c()
    want = [o.cpu() for o in out]
    streams = [torch.cuda.Stream() for _ in q]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, s in zip(calls, streams):
            c(stream=s)
    torch.cuda.synchronize()
    assert all(torch.equal(o.cpu(), w) for o, w in zip(out, want))
