"""The batched serving operators on the GPU against plain float64 forms: appended rows, attention over pages and
over packed prompts, token log probabilities; sizes, masks and layouts where they can go wrong."""
import math

import pytest

torch = pytest.importorskip("torch")

import serving_ref as S  # noqa: E402

pytestmark = pytest.mark.gpu
GPU = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "needs the MI355X"
    from rust_interference_engine_amd import ops
    return ops


def paged(ops, b, window=0, softcap=0.0, scale=None, max_new=None, max_len=None, fill=7.0):
    """outputs of the paged call on the CPU; rows outside the sequences keep `fill`"""
    k, v = b.k_pages.to(GPU), b.v_pages.to(GPU)
    kv = ops.PagedKv(b.paged(k), b.paged(v), b.table.to(GPU))
    seqs = ops.Seqs(b.starts.to(GPU), b.L.to(GPU), max_new=max_new or b.max_new(), max_len=max_len or b.max_len())
    out = torch.full((b.rows, b.H, b.hd), fill, dtype=b.dtype, device=GPU)
    call = ops.PagedAttention(kv, seqs, b.q.to(GPU), out, scale=scale, window=window, softcap=softcap)
    call()
    first = out.cpu()
    call()
    assert torch.equal(out.cpu().nan_to_num(5.0), first.nan_to_num(5.0))  # the same bits again
    return first


def check(b, out, window=0, softcap=0.0, scale=None, fill=7.0):
    scale = 1 / math.sqrt(b.hd) if scale is None else scale
    for i, (n, L) in enumerate(b.lens):
        r = int(b.starts[i])
        q = b.q[r:r + n]
        o, a, size = S.attend(q, b.cached(b.k_pages, i), b.cached(b.v_pages, i), L - n, scale, window, softcap)
        tol = S.tolerance(o, a, size, L, b.hd, b.dtype, softcap)
        err = (out[r:r + n].double() - o).abs()
        assert bool((err <= tol).all()), (i, n, L, float((err / tol).max()))
    assert bool((out[int(b.starts[-1]):] == fill).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,KV,hd", [(4, 1, 32), (15, 5, 64), (14, 2, 64), (6, 6, 96), (8, 2, 128), (8, 1, 128), (4, 1, 256), (3, 1, 256)])
def test_single_tokens(ops, H, KV, hd, dtype):
    b = S.Batch([(1, 1), (1, 17), (1, 32), (1, 33), (1, 0), (1, 500), (0, 64), (1, 129)], H, KV, hd, dtype=dtype, extra_rows=2, extra_cols=1)
    check(b, paged(ops, b))


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("H,KV,hd", [(8, 2, 128), (4, 1, 256), (8, 8, 64)])
@pytest.mark.parametrize("window,softcap", [(0, 0.0), (40, 0.0), (0, 5.0), (1, 2.0)])
def test_a_few_tokens_of_each_sequence(ops, H, KV, hd, page, window, softcap):
    b = S.Batch([(3, 3), (2, 100), (4, 515), (1, 40), (3, 2), (4, 4)], H, KV, hd, page=page, dtype=BF16, seed=1)
    check(b, paged(ops, b, window, softcap), window, softcap)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,KV,hd,page", [(4, 1, 32, 16), (15, 5, 64, 32), (6, 3, 96, 16), (8, 2, 128, 128), (8, 1, 128, 16), (4, 1, 256, 16), (7, 7, 128, 64)])
@pytest.mark.parametrize("window,softcap", [(0, 0.0), (70, 0.0), (0, 3.0)])
def test_chunks_and_single_tokens_in_one_batch(ops, H, KV, hd, page, dtype, window, softcap):
    b = S.Batch([(1, 300), (37, 37), (65, 400), (0, 9), (1, 1), (130, 131), (5, 2)], H, KV, hd, page=page, dtype=dtype, seed=2, extra_rows=3)
    check(b, paged(ops, b, window, softcap), window, softcap)


@pytest.mark.parametrize("lens", [[(1, 5000)], [(2, 4097), (1, 3)], [(40, 6000)], [(1, 4096)] * 3])
@pytest.mark.parametrize("hd", [64, 128])
def test_long_caches_in_splits(ops, lens, hd):
    b = S.Batch(lens, 8, 2, hd, page=64, dtype=F16, seed=3)
    check(b, paged(ops, b))
    check(b, paged(ops, b, 1500), 1500)
    check(b, paged(ops, b, max_len=6000))


def test_rows_of_pages_in_either_order_and_a_scale(ops):
    b = S.Batch([(9, 90), (1, 33)], 8, 4, 64, page=32, seed=4, order="slots")
    check(b, paged(ops, b, scale=0.31), scale=0.31)


def test_large_scores_and_a_moving_maximum(ops):
    b = S.Batch([(1, 700), (60, 700)], 4, 2, 64, seed=5)
    t = b.table[1, :44].long()
    ramp = torch.linspace(0.1, 6.0, 44)[:, None, None, None]  # later keys are ever larger
    b.k_pages[t] = (b.k_pages[t].float() * ramp).half()
    check(b, paged(ops, b))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("H,KV,hd,new", [(8, 2, 128, 60), (8, 2, 64, 3), (4, 1, 256, 40), (4, 1, 256, 2)])
def test_infinite_and_nan_rows_stay_with_the_tokens_that_see_them(ops, H, KV, hd, new, bad):
    L = 200
    b = S.Batch([(new, L), (1, 70)], H, KV, hd, dtype=BF16, seed=6)
    clean = paged(ops, b)
    at = L - 2  # the last two tokens see it
    page, slot = int(b.table[0, at // 16]), at % 16
    b.v_pages[page, 0, slot, 5] = bad
    out = paged(ops, b)
    G = H // KV
    assert torch.equal(out[new:], clean[new:]) and torch.equal(out[:new - 2], clean[:new - 2])
    hit = out[new - 2:new, :G]
    assert bool((hit[..., 5].isnan() if bad != bad else hit[..., 5] == bad).all())
    keep = torch.ones(hd, dtype=torch.bool)
    keep[5] = False
    assert torch.equal(hit[..., keep], clean[new - 2:new, :G][..., keep]) and torch.equal(out[:, G:], clean[:, G:])
    b.v_pages[page, 0, slot, 5] = 0
    b.k_pages[page, 0, slot, 3] = float("nan")  # a key: every number of the tokens that see it
    out = paged(ops, b)
    assert torch.equal(out[:new - 2], clean[:new - 2]) and bool(out[new - 2:new, :G].isnan().all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lens", [[(1, 3000)], [(3, 3000)], [(70, 3000), (1, 2000)]])
def test_an_infinite_value_among_many_makes_that_infinity(ops, dtype, lens):
    """far in a long cache, where all rows see it, with a probability that f16 rounds to zero; whole, and in splits"""
    b = S.Batch(lens, 8, 2, 128, page=64, dtype=dtype, seed=28)
    t = b.table[0, :47].long()
    for p, j in ((20, 1), (30, 2)):
        b.v_pages[t[p], 1, 9, 64 + j] = math.inf if j == 1 else -math.inf
    b.v_pages[t[40], 1, 3, 65 + 1] = math.inf  # dim 66 has both
    b.k_pages[t[20], 1, 9] = -8 * b.q[0, 4].sign()  # hardly seen by one row
    for kw in (dict(), dict(max_len=60000)):
        out = paged(ops, b, **kw)
        n = lens[0][0]
        assert bool((out[:n, 4:, 65] == math.inf).all()) and bool(out[:n, 4:, 66].isnan().all())
        rest = torch.ones(out.shape, dtype=torch.bool)
        rest[:n, 4:, 65:67] = False
        assert bool(torch.isfinite(out[rest]).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lens", [[(1, 3000)], [(3, 3000)], [(70, 3000), (1, 2000)], [(1, 3000)] + [(1, 20)] * 299])
def test_an_infinite_value_of_a_split_that_weighs_nothing(ops, dtype, lens):
    """the first half of the positions scores hundreds below the second for one row: e^-471 or so of their sum"""
    b = S.Batch(lens, 8, 2, 128, page=64, dtype=dtype, seed=41)
    t = b.table[0, :47].long()
    b.k_pages[t[:24], 1] = -40 * b.q[0, 4].sign()
    b.v_pages[t[2], 1, 9, 65] = math.inf
    b.v_pages[t[20], 1, 9, 66] = -math.inf
    for kw in (dict(), dict(max_len=60000)):
        out = paged(ops, b, **kw)
        n = lens[0][0]
        assert bool((out[:n, 4:, 65] == math.inf).all()) and bool((out[:n, 4:, 66] == -math.inf).all())
        rest = torch.ones(out.shape, dtype=torch.bool)
        rest[:n, 4:, 65:67] = False
        assert bool(torch.isfinite(out[rest]).all())


def spoil(v, share, seed):
    """a copy of values v with that share of them infinite or NaN"""
    g = torch.Generator().manual_seed(seed)
    v = v.clone()
    at = torch.rand(v.shape, generator=g) < share
    v[at] = torch.tensor([math.inf, -math.inf, math.nan])[torch.randint(0, 3, (int(at.sum()),), generator=g)].to(v.dtype)
    return v


def spoilt(v, pos0, n, window, H):
    """[n, H, hd]: the sum of the infinite and NaN values that each of n tokens sees, 0 without one"""
    L, KV, hd = v.shape
    seen = []
    for bad in (v.isnan(), v == math.inf, v == -math.inf):
        c = torch.cat([torch.zeros(1, KV, hd), bad.float().cumsum(0)])
        p = pos0 + torch.arange(n)
        hi = (p + 1).clamp(0, L)
        lo = (p + 1 - window).clamp(0, L) if window else torch.zeros_like(p)
        seen.append((c[hi] - c[torch.minimum(lo, hi)]) > 0)
    nan, up, down = seen
    x = torch.where(nan | (up & down), math.nan, torch.where(up, math.inf, torch.where(down, -math.inf, 0.0)))
    return x.repeat_interleave(H // KV, 1)


def check_spoilt(got, q, k, v, pos0, window, dtype, hd):
    n, H = q.shape[:2]
    want = spoilt(v, pos0, n, window, H)
    o, a, size = S.attend(q, k, torch.where(torch.isfinite(v.float()), v, torch.zeros((), dtype=dtype)), pos0, 1 / math.sqrt(hd), window)
    fine = want == 0
    assert torch.equal(got.float()[~fine].nan_to_num(1.0, 2.0, 3.0), want[~fine].float().nan_to_num(1.0, 2.0, 3.0))
    tol = S.tolerance(o, a, size, k.shape[0], hd, dtype)
    assert bool(((got.double() - o).abs() <= tol)[fine].all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("share", [1e-4, 2e-3, 0.3])
@pytest.mark.parametrize("H,KV,hd", [(4, 2, 32), (4, 1, 64), (6, 6, 96), (8, 2, 128), (2, 1, 256)])
@pytest.mark.parametrize("window", [0, 3, 40, 300])
@pytest.mark.parametrize("lens", [[(1, 700), (5, 90), (3, 900), (1, 1)], [(1, 700), (130, 900), (77, 77)]])  # few rows; tiles
def test_infinite_and_nan_values_anywhere(ops, lens, window, H, KV, hd, share, dtype):
    b = S.Batch(lens, H, KV, hd, page=32, dtype=dtype, seed=36)
    b.v_pages = spoil(b.v_pages, share, 37)
    for kw in (dict(), dict(max_len=60000)):  # whole, and in splits
        got = paged(ops, b, window, **kw)
        for i, (n, L) in enumerate(lens):
            r = int(b.starts[i])
            check_spoilt(got[r:r + n], b.q[r:r + n], b.cached(b.k_pages, i), b.cached(b.v_pages, i), L - n, window, dtype, hd)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,KV,hd", [(4, 2, 32), (4, 1, 64), (6, 6, 96), (8, 2, 128), (2, 1, 256)])
@pytest.mark.parametrize("window", [0, 40])
def test_infinite_and_nan_values_anywhere_in_packed_prompts(ops, window, H, KV, hd, dtype):
    lens = [300, 1, 64, 130]
    n = sum(lens)
    g = torch.Generator().manual_seed(38)
    q, k, v = (torch.randn(n, x, hd, generator=g).to(dtype) for x in (H, KV, KV))
    v = spoil(v, 2e-3, 39)
    starts = torch.tensor([0] + lens).cumsum(0).int()
    out = torch.empty(n, H, hd, dtype=dtype, device=GPU)
    ops.PackedAttention(ops.Seqs(starts.to(GPU), max_new=300, max_len=300), q.to(GPU), k.to(GPU), v.to(GPU), out, window=window)()
    for i, L in enumerate(lens):
        r = slice(int(starts[i]), int(starts[i]) + L)
        check_spoilt(out.cpu()[r], q[r], k[r], v[r], 0, window, dtype, hd)


@pytest.mark.parametrize("what", ["first row NaN", "last row NaN", "all NaN", "all infinite"])
@pytest.mark.parametrize("case", ["packed", "chunk", "tokens"])
def test_values_that_are_nan_do_not_stall_a_call(ops, case, what):
    """the positions are searched once for all of a wave's rows: a call takes a few times its time, where a search for every
    output took hundreds"""
    H, KV, hd = 32, 8, 128
    g = torch.Generator(device=GPU).manual_seed(40)
    new, L = {"packed": (3000, 3000), "chunk": (500, 8000), "tokens": (4, 40000)}[case]
    q = torch.randn(new, H, hd, device=GPU, generator=g).to(BF16)
    k, v = (torch.randn(L // 64 + 1, 64, KV, hd, device=GPU, generator=g).to(BF16) for _ in range(2))
    out = torch.empty_like(q)
    starts, lens = torch.tensor([0, new], dtype=torch.int32, device=GPU), torch.tensor([L], dtype=torch.int32, device=GPU)
    seqs = ops.Seqs(starts, lens, max_new=new, max_len=L)
    if case == "packed":
        call = ops.PackedAttention(seqs, q, k.flatten(0, 1)[:L], v.flatten(0, 1)[:L], out)
    else:
        call = ops.PagedAttention(ops.PagedKv(k, v, torch.arange(L // 64 + 1, dtype=torch.int32, device=GPU)[None]), seqs, q, out)

    def time():
        e = [torch.cuda.Event(enable_timing=True) for _ in range(8)]
        for x in e:
            x.record()
            call()
        torch.cuda.synchronize()
        return min(a.elapsed_time(b) for a, b in zip(e[1:], e[2:]))

    clean = time()
    assert bool(torch.isfinite(out).all())
    rows = v.flatten(0, 1)[:L]
    if what == "all infinite":
        rows[:] = math.inf
    else:
        rows[{"first row NaN": slice(0, 1), "last row NaN": slice(L - 1, L), "all NaN": slice(0, L)}[what]] = math.nan
    spoilt_ms = time()
    print(f"{case}, {what}: {clean * 1e3:.0f} us, {spoilt_ms * 1e3:.0f} us")
    sees = torch.arange(new, device=GPU) == new - 1 if what == "last row NaN" else torch.ones(new, dtype=torch.bool, device=GPU)
    assert bool((out[sees] == math.inf).all() if what == "all infinite" else out[sees].isnan().all()) and bool(torch.isfinite(out[~sees]).all())
    assert spoilt_ms < 20 * clean + 1, (clean, spoilt_ms)


def test_slots_behind_the_last_position_may_hold_anything(ops):
    b = S.Batch([(1, 37), (20, 50), (2, 33)], 4, 2, 64, seed=7)
    clean = paged(ops, b)
    for i, (_, L) in enumerate(b.lens):
        page = int(b.table[i, (L - 1) // 16])
        b.k_pages[page, :, (L - 1) % 16 + 1:] = float("nan")
        b.v_pages[page, :, (L - 1) % 16 + 1:] = float("inf")
    assert torch.equal(paged(ops, b), clean)


@pytest.mark.parametrize("new", [1, 50])
def test_positions_of_pages_that_are_none_are_not_seen(ops, new):
    b = S.Batch([(new, 210), (1, 60)], 8, 2, 128, seed=8)
    good = b.table.clone()
    for bad in (-1, b.n_pages, 2 ** 31 - 1, -2 ** 31):
        b.table[0, 3] = bad
        out = paged(ops, b)
        k = torch.cat([b.cached(b.k_pages, 0, 48), b.k_pages.transpose(1, 2)[good[0, 4:].long()].reshape(-1, 2, 128)])[:194]
        v = torch.cat([b.cached(b.v_pages, 0, 48), b.v_pages.transpose(1, 2)[good[0, 4:].long()].reshape(-1, 2, 128)])[:194]
        o, a, size = S.attend(b.q[:new], k, v, 194 - new, 1 / math.sqrt(128))
        tol = S.tolerance(o, a, size, 210, 128, F16)
        assert bool(((out[:new].double() - o).abs() <= tol).all())
        b.table.copy_(good)


def past_the_table(lens, cap, *args, **kw):
    """a batch whose tables address `cap` positions each, with lengths that may pass them"""
    b = S.Batch([(n, cap) for n, _ in lens], *args, **kw)
    b.L = torch.tensor([x for _, x in lens], dtype=torch.int32)
    return b


# (1, 90) and (6, 100) begin past the table; 2^31 - 1 lies behind any window
PAST = [(1, 49), (3, 50), (1, 48), (1, 90), (6, 50), (6, 100), (2, 2 ** 31 - 1)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,KV,hd", [(2, 1, 32), (4, 1, 64), (4, 2, 96), (8, 2, 128), (4, 1, 256)])
@pytest.mark.parametrize("window", [0, 1, 5, 40])
@pytest.mark.parametrize("more", [[], [(70, 52), (30, 49), (20, 90)]])  # with the chunks, the tile kernel
def test_tokens_past_the_table_see_what_it_addresses(ops, more, window, H, KV, hd, dtype):
    lens = PAST + more
    b = past_the_table(lens, 48, H, KV, hd, dtype=dtype, seed=32, extra_rows=1)
    for kw in (dict(), dict(max_len=2 ** 30)):
        got = paged(ops, b, window, **kw)
        for i, (n, L) in enumerate(lens):
            r = int(b.starts[i])
            o, a, size = S.attend(b.q[r:r + n], b.cached(b.k_pages, i), b.cached(b.v_pages, i), L - n, 1 / math.sqrt(hd), window)
            tol = S.tolerance(o, a, size, 48, hd, dtype)
            assert bool(((got[r:r + n].double() - o).abs() <= tol).all()), (i, n, L)
        assert bool((got[-1] == 7).all())


@pytest.mark.parametrize("new", [2, 60])
@pytest.mark.parametrize("window", [2 ** 30, 2 ** 30 + 20, 2 ** 31 - 1])
def test_windows_as_long_as_they_may_be(ops, window, new):
    lens = [(new, 2 ** 30 + 40), (1, 2 ** 31 - 1), (1, 48), (new, 30), (1, 2 ** 30 + 20)]
    b = past_the_table(lens, 48, 8, 2, 64, seed=42)
    got = paged(ops, b, window)
    for i, (n, L) in enumerate(lens):
        r = int(b.starts[i])
        o, a, size = S.attend(b.q[r:r + n], b.cached(b.k_pages, i), b.cached(b.v_pages, i), L - n, 1 / 8, window)
        assert bool(((got[r:r + n].double() - o).abs() <= S.tolerance(o, a, size, 48, 64, F16)).all()), (i, n, L)


@pytest.mark.parametrize("new", [3, 40])
def test_long_tables_that_end_before_the_sequence(ops, new):
    lens = [(new, 3010), (1, 3001), (1, 2900)]
    b = past_the_table(lens, 2944, 8, 2, 64, dtype=BF16, seed=33)
    for window in (0, 700):
        for kw in (dict(), dict(max_len=60000)):
            got = paged(ops, b, window, **kw)
            for i, (n, L) in enumerate(lens):
                r = int(b.starts[i])
                o, a, size = S.attend(b.q[r:r + n], b.cached(b.k_pages, i), b.cached(b.v_pages, i), L - n, 1 / 8, window)
                assert bool(((got[r:r + n].double() - o).abs() <= S.tolerance(o, a, size, 2944, 64, BF16)).all()), (i, n, L)


def test_append_drops_the_tokens_past_the_table(ops):
    lens = [(1, 33), (10, 37), (1, 32), (8, 40), (5, 2 ** 31 - 1), (40, 36), (1, -4)]
    b = past_the_table(lens, 32, 2, 2, 64, seed=34)
    g = torch.Generator().manual_seed(35)
    new = torch.randn(b.rows, 4, 64, generator=g).half()
    dev, k, v = new.to(GPU), b.k_pages.to(GPU), b.v_pages.to(GPU)
    kv = ops.PagedKv(b.paged(k), b.paged(v), b.table.to(GPU))
    ops.PagedAppend(kv, ops.Seqs(b.starts.to(GPU), b.L.to(GPU), max_new=40, max_len=64), dev[:, :2], dev[:, 2:])()
    want_k, want_v = b.paged(b.k_pages).clone(), b.paged(b.v_pages).clone()
    for i, (n, L) in enumerate(lens):
        for t in range(n):
            p = L - n + t
            if 0 <= p < 32:
                at = (int(b.table[i, p // 16]), p % 16)
                want_k[at], want_v[at] = new[int(b.starts[i]) + t, :2], new[int(b.starts[i]) + t, 2:]
    assert torch.equal(b.paged(k.cpu()), want_k) and torch.equal(b.paged(v.cpu()), want_v)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,KV,hd", [(4, 2, 32), (15, 5, 64), (4, 4, 96), (8, 2, 128), (8, 1, 128), (4, 1, 256)])
@pytest.mark.parametrize("window,softcap", [(0, 0.0), (50, 0.0), (0, 4.0)])
def test_packed_prompts(ops, H, KV, hd, dtype, window, softcap):
    lens = [1, 64, 0, 129, 33, 300, 2, 128]
    g = torch.Generator().manual_seed(9)
    n = sum(lens)
    qkv = torch.randn(n + 2, H + 2 * KV, hd, generator=g).to(dtype)
    dev = qkv.to(GPU)
    starts = torch.tensor([0] + lens).cumsum(0).int()
    out = torch.full((n + 2, H + 1, hd), 3.0, dtype=dtype, device=GPU)[:, :H]
    call = ops.PackedAttention(ops.Seqs(starts.to(GPU), max_new=max(lens), max_len=max(lens)), dev[:, :H], dev[:, H:H + KV], dev[:, H + KV:],
                               out, window=window, softcap=softcap)
    call()
    got = out.cpu()
    for i, L in enumerate(lens):
        r = int(starts[i])
        if not L:
            continue
        o, a, size = S.attend(qkv[r:r + L, :H], qkv[r:r + L, H:H + KV], qkv[r:r + L, H + KV:], 0, 1 / math.sqrt(hd), window, softcap)
        tol = S.tolerance(o, a, size, L, hd, dtype, softcap)
        assert bool(((got[r:r + L].double() - o).abs() <= tol).all()), (i, L)
    assert bool((got[n:] == 3).all())


def test_one_long_prompt_in_splits(ops):
    g = torch.Generator().manual_seed(10)
    L, H, KV, hd = 1500, 4, 1, 128
    q, k, v = (torch.randn(L, x, hd, generator=g).half() for x in (H, KV, KV))
    out = torch.empty(L, H, hd, dtype=F16, device=GPU)
    ops.PackedAttention(ops.Seqs(torch.tensor([0, L], dtype=torch.int32, device=GPU), max_new=L, max_len=L), q.to(GPU), k.to(GPU), v.to(GPU), out)()
    o, a, size = S.attend(q, k, v, 0, 1 / math.sqrt(hd))
    assert bool(((out.cpu().double() - o).abs() <= S.tolerance(o, a, size, L, hd, F16)).all())


@pytest.mark.parametrize("n_seq", [1, 63, 64, 65, 200, 4100])
def test_many_sequences(ops, n_seq):
    lens = [(i % 3, max(1, i % 40)) for i in range(n_seq)]
    b = S.Batch(lens, 2, 1, 32, seed=11, extra_rows=1)  # one sequence, no token: a batch of none is refused
    out = paged(ops, b)
    got = paged(ops, b, max_new=40)  # the tile kernel's way
    for i in list(range(0, n_seq, max(1, n_seq // 50))) + [n_seq - 1]:
        n, L = lens[i]
        r = int(b.starts[i])
        o, a, size = S.attend(b.q[r:r + n], b.cached(b.k_pages, i), b.cached(b.v_pages, i), L - n, 1 / math.sqrt(32))
        tol = S.tolerance(o, a, size, L, 32, F16)
        assert bool(((out[r:r + n].double() - o).abs() <= tol).all()) and bool(((got[r:r + n].double() - o).abs() <= tol).all())


@pytest.mark.parametrize("src", [F32, F16, BF16])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("order", ["heads", "slots"])
def test_append(ops, src, dtype, order):
    if src not in (F32, dtype):
        pytest.skip("refused: another 16-bit type")
    lens = [(1, 1), (20, 20), (3, 200), (0, 17), (5, 3), (1, 64)]
    b = S.Batch(lens, 4, 3, 64, dtype=dtype, order=order, extra_rows=2, seed=12)
    g = torch.Generator().manual_seed(13)
    new = torch.randn(b.rows, 6, 64, generator=g).to(src)
    dev, k, v = new.to(GPU), b.k_pages.to(GPU), b.v_pages.to(GPU)
    kv = ops.PagedKv(b.paged(k), b.paged(v), b.table.to(GPU))
    ops.PagedAppend(kv, ops.Seqs(b.starts.to(GPU), b.L.to(GPU), max_new=20, max_len=200), dev[:, :3], dev[:, 3:])()
    want_k, want_v = b.paged(b.k_pages).clone(), b.paged(b.v_pages).clone()
    for i, (n, L) in enumerate(lens):
        for t in range(n):
            p = L - n + t
            if p >= 0:
                at = (int(b.table[i, p // 16]), p % 16)
                want_k[at], want_v[at] = new[int(b.starts[i]) + t, :3].to(dtype), new[int(b.starts[i]) + t, 3:].to(dtype)
    assert torch.equal(b.paged(k.cpu()), want_k) and torch.equal(b.paged(v.cpu()), want_v)


def test_append_leaves_pages_that_are_none_alone(ops):
    b = S.Batch([(40, 40)], 2, 1, 32, seed=14)
    b.table[0, 1] = -5
    k, v = b.k_pages.to(GPU), b.v_pages.to(GPU)
    new = torch.randn(40, 1, 32, device=GPU)
    ops.PagedAppend(ops.PagedKv(b.paged(k), b.paged(v), b.table.to(GPU)), ops.Seqs(b.starts.to(GPU), b.L.to(GPU), max_new=40, max_len=40), new, new)()
    want = b.k_pages.clone()
    want[int(b.table[0, 0]), 0] = new[:16, 0].half().cpu()
    want[int(b.table[0, 2]), 0, :8] = new[32:, 0].half().cpu()
    assert torch.equal(k.cpu(), want)


# ln p of f32 logits, all within R of each other: x − m and the two subtractions round to 2^-24 of at most R each, ln S is
# off by the sum's n·2^-24 at most (chains are far shorter), an exponential by 2^-22 + R·2^-23
def logprob_tol(x, V):
    fin = x[torch.isfinite(x)]
    R = float(fin.max() - fin.min()) if fin.numel() else 0.0
    return 3 * (R + math.log(V) + 1) * 2.0 ** -24 + (V / 64 + 40) * 2.0 ** -24 + 2.0 ** -21 + min(R, 40.0) * 2.0 ** -22


def run_logprobs(ops, x, targets, top):
    n, V = x.shape
    lp, h = torch.full((n,), 9.0, device=GPU), torch.full((n,), 9.0, device=GPU)
    ids = torch.full((n, top), -9, dtype=torch.int32, device=GPU) if top else None
    tops = torch.full((n, top), 9.0, device=GPU) if top else None
    ops.TokenLogprobs(x, targets=targets.to(GPU), logprob=lp, entropy=h, top_ids=ids, top_logprobs=tops)()
    return lp.cpu().double(), h.cpu().double(), ids.cpu() if top else None, tops.cpu().double() if top else None


def check_logprobs(ops, x, dev, targets, top):
    lp, h, ids, tops = run_logprobs(ops, dev, targets, top)
    wl, wh, wi, wt = S.logprobs(x, targets, top)
    tol = logprob_tol(x.double(), x.shape[1])

    def near(a, b, t):
        fine = torch.isfinite(b)
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a[~fine].nan_to_num(1.0, 2.0, 3.0), b[~fine].nan_to_num(1.0, 2.0, 3.0))
        assert bool(((a - b).abs()[fine] <= t).all()), float((a - b).abs()[fine].max() / t)

    near(lp, wl, tol)
    near(h, wh, tol * (1 + 2 * math.log(x.shape[1])))  # ln S, and a mean of x − m over the same probabilities
    if top:
        assert torch.equal(ids.long(), wi)
        near(tops, wt, tol)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("V,n,top", [(1, 2, 1), (5, 3, 5), (511, 4, 3), (512, 3, 20), (513, 2, 64), (1100, 3, 64), (40007, 5, 20), (49152, 9, 1), (151936, 2, 5)])
def test_logprobs(ops, V, n, top, dtype):
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(n, V, generator=g) * 3).to(dtype)
    t = torch.randint(0, V, (n,), generator=g).int()
    t[0] = V if n > 2 else t[0]  # no token
    check_logprobs(ops, x, x.to(GPU), t, top)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("off", [1, 3, 7])
def test_logprobs_of_rows_at_any_place(ops, dtype, off):
    g = torch.Generator().manual_seed(off)
    x = torch.randn(3, 3001, generator=g).to(dtype)
    dev = torch.full((3, 3100), 50.0, dtype=dtype, device=GPU)  # its neighbours would win
    dev[:, off:off + 3001] = x.to(GPU)
    check_logprobs(ops, x, dev[:, off:off + 3001], torch.tensor([0, 3000, -1], dtype=torch.int32), 20)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_logprobs_of_odd_rows(ops, dtype):
    inf, nan, low = math.inf, math.nan, torch.finfo(dtype).min
    V = 5000
    g = torch.Generator().manual_seed(3)
    x = torch.randn(10, V, generator=g)
    x[0] = 2.5                     # all equal: the lowest indices
    x[1, :4990] = -inf             # nearly all masked
    x[2] = -inf                    # nothing
    x[3, 77] = nan
    x[4, 4000] = inf
    x[5, 100:] = low               # masks of the lowest value
    x[6] = -inf
    x[6, 3] = 0                    # one token
    x[7] = 0
    x[7, 10:3000] = 1              # more ties than are ranked at once
    x[8] = nan
    x[9] = low
    x = x.to(dtype)
    t = torch.tensor([0, 4995, 1, 2, 4000, 200, 3, 10, 0, 9], dtype=torch.int32)
    lp, h, ids, tops = run_logprobs(ops, x.to(GPU), t, 20)
    wl, wh, wi, wt = S.logprobs(x, t, 20)
    wi = wi.long()
    for r in range(10):
        assert torch.equal(ids[r].long(), wi[r]), r
        tol = 2.0 ** -18 * (1 + math.log(V)) ** 2
        for a, b in ((lp[r:r + 1], wl[r:r + 1]), (h[r:r + 1], wh[r:r + 1]), (tops[r], wt[r])):
            assert torch.equal(a.isnan(), b.isnan()), r
            fine = torch.isfinite(b)
            big = fine & (b.abs() > 1e4)  # a masked token's own: the difference of two logits, to a step
            assert bool(((a - b).abs()[fine & ~big] <= tol).all()), r
            assert bool(((a - b).abs()[big] <= b.abs()[big] * 2.0 ** -22).all()), r
            assert torch.equal(a[~fine & ~b.isnan()], b[~fine & ~b.isnan()]), r


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n", [6, 2001])  # 2001 rows: runs of more than one group
@pytest.mark.parametrize("mag", [6e4, 1e6, 1.1e6, 3e7, 1e9, 5e9, 1e10, 1e12, 1e15, 1e20, 1e25, 1e29, 3e30, 3e38])
def test_logprobs_of_large_finite_logits(ops, mag, n, dtype):
    """masks and logits of any finite size: whole runs of them, single ones, and rows of nothing else"""
    if mag > torch.finfo(dtype).max:
        mag = 6e4
    V = 20016
    g = torch.Generator().manual_seed(31)
    x = torch.randn(6, V, generator=g) * 3
    x[0, 3000:9000] = -mag            # runs of groups that hold nothing else
    x[1, 777] = -mag                  # one masked
    x[2, 12345] = mag                 # one that takes all
    x[3] = x[3] + mag                 # all large, as far apart as their steps let them
    x[4] = x[4] - mag
    x[5, :] = -mag
    x[5, 4000] = 1.5                  # all masked but one
    x = x.to(dtype)
    x[3:5] = x[3:5].clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max)
    t = torch.tensor([5, 777, 12345, 9, 10, 4000], dtype=torch.int32)
    rep = -(-n // 6)
    lp, h, ids, tops = run_logprobs(ops, x.repeat(rep, 1)[:n].to(GPU), t.repeat(rep)[:n], 4)
    for a in (lp, h, ids, tops):
        assert torch.equal(a, torch.cat([a[:6]] * rep)[:n])
    wl, wh, wi, wt = S.logprobs(x, t, 4)
    assert torch.equal(ids[:6].long(), wi)
    for r in range(6):
        row = x[r].double()
        near = row[row > row.max() - 200]  # the others' probabilities are zeros in f32
        tol = logprob_tol(near, V)
        for a, b, tl in ((lp[r:r + 1], wl[r:r + 1], tol), (h[r:r + 1], wh[r:r + 1], tol * (1 + 2 * math.log(V))), (tops[r], wt[r], tol)):
            # two differences of numbers of the size of b, each rounded once: 2 * 2^-24 |b|
            assert bool(((a - b).abs() <= tl + b.abs() * 2.0 ** -23).all()), (r, a, b)


def test_logprobs_of_a_nearly_certain_token(ops):
    x = torch.zeros(1, 4000)
    x[0, 1234] = 30.0
    lp, h, _, _ = run_logprobs(ops, x.to(GPU), torch.tensor([1234], dtype=torch.int32), 0)
    rest = 3999 * math.exp(-30)  # −ln p = ln(1 + rest), H = ln(1 + rest) + 30 rest / (1 + rest): 3.7e-10 and 1.2e-8 keep their digits
    assert abs(float(lp[0]) / -math.log1p(rest) - 1) < 1e-5 and abs(float(h[0]) / (math.log1p(rest) + 30 * rest / (1 + rest)) - 1) < 1e-5


def test_a_step_of_a_batch_captured_and_replayed(ops):
    """append, attention over the pages, log probabilities of rows made from its outputs: as one graph over buffers
    that change between the replays, on a stream of its own"""
    b = S.Batch([(1, 90), (7, 60), (1, 1), (1, 2100)], 8, 2, 64, seed=15)
    g = torch.Generator().manual_seed(16)
    k, v = b.k_pages.to(GPU), b.v_pages.to(GPU)
    kv = ops.PagedKv(b.paged(k), b.paged(v), b.table.to(GPU))
    seqs = ops.Seqs(b.starts.to(GPU), b.L.to(GPU), max_new=7, max_len=2100)
    new = torch.empty(b.rows, 4, 64, device=GPU)
    q, out = torch.empty(b.rows, 8, 64, dtype=F16, device=GPU), torch.empty(b.rows, 8, 64, dtype=F16, device=GPU)
    logits = out.view(b.rows, 512)
    t = torch.arange(b.rows, dtype=torch.int32, device=GPU)
    lp, h = torch.empty(b.rows, device=GPU), torch.empty(b.rows, device=GPU)
    calls = [ops.PagedAppend(kv, seqs, new[:, :2], new[:, 2:]), ops.PagedAttention(kv, seqs, q, out), ops.TokenLogprobs(logits, targets=t, logprob=lp, entropy=h)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        for c in calls:
            c()
    for rep in range(4):
        new.copy_(torch.randn(b.rows, 4, 64, generator=g))
        q.copy_(torch.randn(b.rows, 8, 64, generator=g))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = out.cpu().clone(), lp.cpu().clone(), h.cpu().clone(), k.cpu().clone()
        for x in (out, lp, h):
            x.zero_()
        for c in calls:
            c(stream=side if rep % 2 else None)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y.cpu()) for x, y in zip(got, (out, lp, h, k)))
        b.k_pages, b.v_pages, b.q = k.cpu(), v.cpu(), q.cpu()
        r, n, L = int(b.starts[1]), 7, 60
        assert torch.equal(b.cached(b.k_pages, 1)[L - n:], new[r:r + n, :2].half().cpu())
        check(b, out.cpu())


def test_two_calls_at_once_on_two_streams(ops):
    a = S.Batch([(1, 3000), (1, 500)], 8, 2, 128, seed=17)
    b = S.Batch([(2, 2500)], 8, 2, 128, seed=18)
    alone = [paged(ops, x) for x in (a, b)]
    made = []
    for x in (a, b):
        kv = ops.PagedKv(x.paged(x.k_pages.to(GPU)), x.paged(x.v_pages.to(GPU)), x.table.to(GPU))
        out = torch.zeros(x.rows, 8, 128, dtype=F16, device=GPU)
        made.append((ops.PagedAttention(kv, ops.Seqs(x.starts.to(GPU), x.L.to(GPU), max_new=x.max_new(), max_len=x.max_len()), x.q.to(GPU), out), out, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        for call, out, st in made:
            call(stream=st)
    torch.cuda.synchronize()
    for (_, out, _), want in zip(made, alone):
        assert torch.equal(out.cpu(), want)


@pytest.mark.parametrize("H,KV,new", [(40, 1, 1), (71, 1, 3), (33, 1, 1), (256, 2, 2), (32, 1, 1), (17, 1, 1)])
def test_many_query_heads_on_one_kv_head(ops, H, KV, new):
    b = S.Batch([(new, 150), (new, new), (1, 700)], H, KV, 64, dtype=BF16, seed=21)
    check(b, paged(ops, b))


def test_the_first_sequence_may_start_behind_other_rows(ops):
    b = S.Batch([(5, 70), (40, 300), (1, 9)], 8, 2, 64, seed=22)
    shift = 37
    b.q = torch.cat([torch.full((shift, 8, 64), math.nan, dtype=F16), b.q])
    b.starts += shift
    b.rows += shift
    for kw in (dict(), dict(max_len=20000)):  # without and with splits
        out = paged(ops, b, **kw)
        assert bool((out[:shift] == 7).all())
        check(b, out)
    g = torch.Generator().manual_seed(23)
    new = torch.randn(b.rows, 2, 64, generator=g).half()
    k, v, dev = b.k_pages.to(GPU), b.v_pages.to(GPU), new.to(GPU)
    ops.PagedAppend(ops.PagedKv(b.paged(k), b.paged(v), b.table.to(GPU)), ops.Seqs(b.starts.to(GPU), b.L.to(GPU), max_new=40, max_len=300), dev, dev)()
    b.k_pages = k.cpu()
    assert torch.equal(b.cached(b.k_pages, 1)[-40:], new[shift + 5:shift + 45]) and torch.equal(b.cached(b.k_pages, 2)[-1:], new[-1:])


@pytest.mark.parametrize("new", [1, 3, 60])
@pytest.mark.parametrize("hd", [128, 256])
def test_pages_below_the_window_may_be_gone(ops, new, hd):
    b = S.Batch([(new, 400), (1, 333)], 4, 1, hd, dtype=BF16, seed=24)
    whole = paged(ops, b, 100)
    check(b, whole, 100)
    for i, (n, L) in enumerate(b.lens):
        gone = (L - n - 99) // 16  # pages that no token's window reaches
        b.table[i, :gone] = torch.tensor([-1, 2 ** 31 - 1, b.n_pages])[torch.arange(gone) % 3].int()
        page = int(b.table[i, gone])
        b.v_pages[page, :, :(L - n - 99) % 16] = math.nan  # and the slots of the last page that it only ends in
        b.k_pages[page, :, :(L - n - 99) % 16] = math.inf
    assert torch.equal(paged(ops, b, 100), whole)


@pytest.mark.parametrize("new", [2, 50])
def test_a_query_that_is_nan_or_infinite_spoils_its_own_row_only(ops, new):
    b = S.Batch([(new, 130), (1, 50)], 8, 2, 64, seed=25)
    clean = paged(ops, b)
    b.q[1, 3, 7], b.q[new, 0, 0] = math.nan, math.inf
    out = paged(ops, b)
    assert bool(out[1, 3].isnan().all()) and bool((~torch.isfinite(out[new, 0])).all())
    out[1, 3], out[new, 0] = clean[1, 3], clean[new, 0]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
def test_packed_prompts_keep_infinite_and_nan_values_to_the_tokens_behind_them(ops, hd):
    lens, H, KV = [70, 40, 90], 4, 2
    g = torch.Generator().manual_seed(26)
    q, k, v = (torch.randn(200, x, hd, generator=g).to(BF16) for x in (H, KV, KV))
    starts = torch.tensor([0] + lens).cumsum(0).int().to(GPU)

    def run():
        out = torch.empty(200, H, hd, dtype=BF16, device=GPU)
        ops.PackedAttention(ops.Seqs(starts, max_new=90, max_len=90), q.to(GPU), k.to(GPU), v.to(GPU), out)()
        return out.cpu()

    clean = run()
    v[70 + 17, 1, 2], v[69, 0, 0], v[110, 0, hd - 1] = math.inf, math.nan, -math.inf
    out = run()
    hit = torch.zeros(200, H, hd, dtype=torch.bool)
    hit[70 + 17:110, 2:, 2] = True   # of sequence 1, behind its token 17, heads of KV head 1
    hit[69, :2, 0] = True            # the last token of sequence 0
    hit[110:, :2, hd - 1] = True     # all of sequence 2
    assert torch.equal(out[~hit], clean[~hit])
    assert bool((out[70 + 17:110, 2:, 2] == math.inf).all()) and bool(out[69, :2, 0].isnan().all()) and bool((out[110:, :2, hd - 1] == -math.inf).all())


@pytest.mark.parametrize("sign", [False, True])
@pytest.mark.parametrize("lens", [[(1, 3000), (3, 77)], [(1, 3000), (60, 700)]])  # few rows; tiles
@pytest.mark.parametrize("hd", [64, 256])
def test_values_as_large_as_the_type_holds(ops, hd, lens, sign):
    b = S.Batch(lens, 4, 2, hd, page=64, dtype=BF16, seed=49)
    big = torch.finfo(BF16).max
    b.v_pages = (torch.where(b.v_pages < 0, -1.0, 1.0) * big).to(BF16) if sign else torch.full_like(b.v_pages, big)
    for kw in (dict(), dict(max_len=60000)):
        got = paged(ops, b, **kw)
        check(b, got)
        assert bool(torch.isfinite(got).all())


@pytest.mark.parametrize("lens", [[(1, 3000), (3, 77)], [(1, 3000), (60, 700)]])  # few rows; tiles
@pytest.mark.parametrize("power", [-40, -70, -80])
def test_small_values_keep_their_digits(ops, power, lens):
    b = S.Batch(lens, 4, 2, 64, page=64, dtype=BF16, seed=50)
    b.v_pages = (b.v_pages.double() * 2.0 ** power).to(BF16)
    for kw in (dict(), dict(max_len=60000)):
        # terms under 2^-126 may be lost, 2^-94 of the values' weights of one
        check(b, paged(ops, b, **kw))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lens", [[(1, 3000), (3, 77)], [(1, 3000), (60, 700)]])  # few rows; tiles
def test_keys_of_minus_infinity_have_no_weight(ops, lens, dtype):
    b = S.Batch(lens, 4, 2, 64, page=64, dtype=dtype, seed=51)
    b.q[..., 0] = b.q[..., 0].abs() + 0.5
    keys = b.paged(b.k_pages)
    keep = [(0, 2990), (0, 100), (1, 10), (1, 70)]  # of sequence and position; KV head 1 has none
    values = keys[..., 0].clone()
    keys[..., 0] = -math.inf
    for i, j in keep:
        at = int(b.table[i, j // 64]), j % 64, 0
        keys[at][0] = values[at]
    for kw in (dict(), dict(max_len=60000)):
        got = paged(ops, b, **kw)
        for i, (n, L) in enumerate(lens):
            r = int(b.starts[i])
            mine = [j for e, j in keep if e == i]
            k, v = b.cached(b.k_pages, i), b.cached(b.v_pages, i)
            for t in range(n):
                see = [j for j in mine if j <= L - n + t]
                assert bool((got[r + t, 2:] == 0).all())  # nothing above -inf: zeros
                if not see:
                    assert bool((got[r + t] == 0).all())
                    continue
                o, a, size = S.attend(b.q[r + t:r + t + 1, :2], k[see, :1], v[see, :1], len(see) - 1, 1 / 8)
                assert bool(((got[r + t, :2].double() - o[0]).abs() <= S.tolerance(o, a, size, L, 64, dtype)[0]).all())


@pytest.mark.parametrize("new", [2, 40])  # few rows; tiles
def test_offsets_past_four_gigabytes(ops, new):
    """pages, rows of queries, of outputs and of packed prompts, and logits, far apart in buffers of 5 GB and more"""
    KV, G, hd, page = 2, 4, 64, 16
    b = S.Batch([(new, 100), (1, 40)], KV * G, KV, hd, page=page, dtype=BF16, seed=52)
    want = paged(ops, b)
    far = 5 * 2 ** 30 // (page * KV * hd * 2)  # that many pages behind
    spread = [torch.empty(far + b.n_pages, KV, page, hd, dtype=BF16, device=GPU) for _ in range(2)]
    for x, y in zip(spread, (b.k_pages, b.v_pages)):
        x[far:] = y.to(GPU)
    last = spread[0][far:].clone()
    step = 2 ** 25  # values from one row to the next: 64 MB, the largest
    rows = b.rows
    wide = torch.empty(rows * step, dtype=BF16, device=GPU)  # 40 new: 2.7 GB
    q, out = wide.as_strided((rows, KV * G, hd), (step, hd, 1)), wide.as_strided((rows, KV * G, hd), (step, hd, 1), 4096)
    q[:] = b.q.to(GPU)
    kv = ops.PagedKv(*(x.transpose(1, 2) for x in spread), (b.table.long().clamp(max=b.n_pages - 1) + far).int().to(GPU))
    seqs = ops.Seqs(b.starts.to(GPU), b.L.to(GPU), max_new=new, max_len=100)
    ops.PagedAttention(kv, seqs, q, out)()
    assert torch.equal(out.cpu(), want)
    k = wide.as_strided((rows, KV, hd), (step, hd, 1), 8192)
    k[:] = torch.randn(rows, KV, hd, device=GPU)
    ops.PagedAppend(kv, seqs, k, k)()
    b.k_pages = spread[0][far:].cpu()
    assert torch.equal(b.cached(b.k_pages, 0)[-new:], k[:new].cpu()) and torch.equal(b.cached(b.k_pages, 1)[-1:], k[new:].cpu())
    assert int((spread[0][far:] != last).any(-1).sum()) == rows * KV  # and nothing else
    del spread, kv, wide, q, out, k

    n = 2 * 64 + 5  # rows behind 4 GB and the first ones
    wide = torch.empty((n - 1) * step + 16384, dtype=F16, device=GPU)
    view = lambda heads, at: wide.as_strided((n, heads, hd), (step, hd, 1), at)  # noqa: E731
    q, k, v, out = view(4, 0), view(2, 1024), view(2, 2048), view(4, 4096)
    for x in (q, k, v):
        x[:] = torch.randn(x.shape, device=GPU)
    starts = torch.tensor([0, 70, n], dtype=torch.int32, device=GPU)
    ops.PackedAttention(ops.Seqs(starts, max_new=70, max_len=70), q, k, v, out)()
    for r in (slice(0, 70), slice(70, n)):
        o, a, size = S.attend(q[r].cpu(), k[r].cpu(), v[r].cpu(), 0, 1 / 8)
        assert bool(((out[r].cpu().double() - o).abs() <= S.tolerance(o, a, size, 70, hd, F16)).all())
    x = wide.as_strided((n, 3001), (step, 1), 8192)
    x[:] = torch.randn(x.shape, device=GPU)
    check_logprobs(ops, x.cpu(), x, torch.arange(n, dtype=torch.int32), 5)


# query heads of a KV head and new tokens: 16 rows (one block), 17 and up to 32 (two), 33 (tiles)
ROWS = [(4, 4), (17, 1), (3, 6), (5, 6), (8, 4), (1, 32), (11, 3)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("G,new", ROWS)
@pytest.mark.parametrize("window,softcap", [(0, 0.0), (40, 0.0), (0, 5.0), (7, 3.0)])
def test_sixteen_to_thirty_three_rows_of_a_sequence(ops, G, new, hd, window, softcap, dtype):
    b = S.Batch([(new, 700), (new, new), (1, 45), (new, 300), (new, new - 1), (0, 30)], 2 * G, 2, hd, page=32, dtype=dtype, seed=46, extra_rows=1)
    for kw in (dict(), dict(max_len=60000)):  # whole, and in splits
        check(b, paged(ops, b, window, softcap, **kw), window, softcap)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("G,new", ROWS)
@pytest.mark.parametrize("window", [0, 40])
def test_sixteen_to_thirty_three_rows_with_odd_values_and_pages(ops, G, new, hd, window, dtype):
    lens = [(new, 700), (new, 90), (1, 45)]
    b = S.Batch(lens, 2 * G, 2, hd, page=16, dtype=dtype, seed=47)
    b.v_pages = spoil(b.v_pages, 2e-3, 48)
    for kw in (dict(), dict(max_len=60000)):
        got = paged(ops, b, window, **kw)
        for i, (n, L) in enumerate(lens):
            r = int(b.starts[i])
            check_spoilt(got[r:r + n], b.q[r:r + n], b.cached(b.k_pages, i), b.cached(b.v_pages, i), L - n, window, dtype, hd)
    # a page that is none: its 16 positions are not seen, which is as if they lay below a window of their own
    good = b.table.clone()
    for at in (0, 20):
        for bad in (-1, b.n_pages):
            b.table[0, at] = bad
            got = paged(ops, b, 0)
            k, v = (torch.cat([x[:16 * at], x[16 * at + 16:]]) for x in (b.paged(p)[good[0].long().clamp(0, b.n_pages - 1)].reshape(-1, 2, hd)[:700] for p in (b.k_pages, b.v_pages)))
            check_spoilt(got[:new], b.q[:new], k, v, 684 - new, 0, dtype, hd)
            b.table.copy_(good)


@pytest.mark.parametrize("softcap", [1e-38, 1e-3, 0.5, 30.0, 50.0, 1e3, 1e5, 1e7, 1e12, 1e30, 3e38])
@pytest.mark.parametrize("lens", [[(1, 300), (3, 77)], [(1, 300), (60, 100)]])  # few rows; tiles
def test_softcaps_of_any_size(ops, lens, softcap):
    b = S.Batch(lens, 8, 2, 64, dtype=F16, seed=44)
    b.q *= 4  # scores of up to 30 or so
    scale = 1 / 8
    got = paged(ops, b, softcap=softcap)
    for i, (n, L) in enumerate(b.lens):
        r = int(b.starts[i])
        q, k = b.q[r:r + n], b.cached(b.k_pages, i)
        o, a, size = S.attend(q, k, b.cached(b.v_pages, i), L - n, scale, 0, softcap)
        # a capped score is off by 2^-21 of the cap where it is a fifth of it at least, and by a few steps of its own size
        # below that: 2^-19 of the score itself in any case, next to the score's own error, which the cap only makes smaller
        s = q.double().transpose(0, 1) @ k.double().transpose(0, 1).repeat_interleave(4, 0).transpose(1, 2) * scale
        top = float((softcap * torch.tanh(s / softcap)).abs().max())
        tol = S.tolerance(o, a, size, L, 64, F16) + 2 * 2.0 ** -19 * top * a
        err = (got[r:r + n].double() - o).abs()
        assert bool((err <= tol).all()), (i, float((err / tol).max()))


def test_a_workspace_waits_for_what_its_memory_was_used_by(ops):
    """made from memory that the stream it was made on still writes, and called on another one: eagerly, in a capture, and
    made within one"""
    b = S.Batch([(1, 3000), (1, 500)], 8, 2, 128, seed=45)
    want = paged(ops, b)
    kv = ops.PagedKv(b.paged(b.k_pages.to(GPU)), b.paged(b.v_pages.to(GPU)), b.table.to(GPU))
    seqs = ops.Seqs(b.starts.to(GPU), b.L.to(GPU), max_new=1, max_len=3000)
    q, out = b.q.to(GPU), torch.zeros(b.rows, 8, 128, dtype=F16, device=GPU)
    size = ops.PagedAttention(kv, seqs, q, out).workspace.numel()
    a = torch.randn(8192, 8192, device=GPU).half()
    a @ a
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    junk = torch.empty(size, dtype=torch.uint8, device=GPU)
    at = junk.data_ptr()
    x = a
    for _ in range(30):  # some 30 ms
        x = x @ a
    junk.fill_(255)
    written = torch.cuda.current_stream().record_event()
    del junk
    call = ops.PagedAttention(kv, seqs, q, out)
    same = call.workspace.data_ptr() == at
    call(stream=side)
    side.synchronize()
    assert written.query() or not same
    assert same and torch.equal(out.cpu(), want)
    out.zero_()
    torch.cuda.synchronize()
    call(stream=side)  # not again
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    assert torch.equal(out.cpu(), want)

    graph = torch.cuda.CUDAGraph()
    late = ops.PagedAttention(kv, seqs, q, out)
    with torch.cuda.graph(graph, stream=side):
        late()
        inner = ops.PagedAttention(kv, seqs, q, out)
        inner()
        other = torch.cuda.Stream()
        other.wait_stream(side)
        inner(stream=other)
        side.wait_stream(other)
    for _ in range(3):
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.cpu(), want)
        out.zero_()
        late(stream=side)
        side.synchronize()
        assert torch.equal(out.cpu(), want)


def test_strides_of_dimensions_with_one_entry_mean_nothing(ops):
    """one KV head, one row, one page: views whose strides there are odd, far too large or different"""
    g = torch.Generator(device=GPU).manual_seed(43)
    i32 = dict(dtype=torch.int32, device=GPU)
    mk = lambda *shape: torch.randn(*shape, device=GPU, generator=g).half()  # noqa: E731
    n, hd = 30, 64
    k, v = mk(n, hd), mk(n, hd)
    heads = [k.as_strided((n, 1, hd), (hd, 7, 1)), v.as_strided((n, 1, hd), (hd, 1 << 40, 1))]
    plain = [k.view(n, 1, hd), v.view(n, 1, hd)]
    q = mk(n, 2, hd)
    prompts = ops.Seqs(torch.tensor([0, n], **i32), max_new=n, max_len=n)
    outs = []
    for kk, vv in (heads, plain):
        outs.append(torch.empty_like(q))
        ops.PackedAttention(prompts, q, kk, vv, outs[-1])()
    assert torch.equal(*outs)

    pages = [[mk(2, 16, 1, hd), mk(2, 16, 1, hd)] for _ in range(1)] * 2
    table = torch.tensor([[1, 0]], **i32)
    kept = []
    for i, (kk, vv) in enumerate((heads, plain)):
        pk, pv = (x.clone() for x in pages[i])
        if i == 0:
            pk, pv = pk.as_strided(pk.shape, (16 * hd, hd, 3, 1)), pv.as_strided(pv.shape, (16 * hd, hd, 1 << 50, 1))
        kv = ops.PagedKv(pk, pv, table)
        seqs = ops.Seqs(torch.tensor([0, n], **i32), torch.tensor([n], **i32), max_new=n, max_len=32)
        ops.PagedAppend(kv, seqs, kk, vv)()
        one = ops.Seqs(torch.tensor([0, 1], **i32), torch.tensor([n], **i32), max_new=1, max_len=32)
        q1 = mk(1, 2, hd) if i == 0 else q1
        out = torch.empty(200, dtype=F16, device=GPU).as_strided((1, 2, hd), (13, hd, 1)) if i == 0 else torch.empty(1, 2, hd, dtype=F16, device=GPU)
        ops.PagedAttention(kv, one, q1.as_strided((1, 2, hd), (5, hd, 1)) if i == 0 else q1, out)()
        kept.append((pk.reshape(-1).clone(), pv.reshape(-1).clone(), out.reshape(-1).clone()))
    assert all(torch.equal(a, b) for a, b in zip(*kept))
    assert torch.equal(kept[0][0].view(2, 16, hd)[1], k[:16]) and torch.equal(kept[0][1].view(2, 16, hd)[0, :14], v[16:])

    page = mk(1, 16, 2, hd)  # one page
    a = ops.PagedKv(page.as_strided(page.shape, (9, 2 * hd, hd, 1)), page.clone().as_strided(page.shape, (1 << 45, 2 * hd, hd, 1)), torch.zeros(1, 1, **i32))
    out = torch.empty(1, 2, hd, dtype=F16, device=GPU)
    ops.PagedAttention(a, ops.Seqs(torch.tensor([0, 1], **i32), torch.tensor([1], **i32), max_new=1, max_len=16), q[:1], out)()
    assert torch.equal(out[0], page[0, 0])  # of one position its value


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_logprobs_where_every_group_counts(ops, dtype):
    """vocabularies past the registers' groups, equal maxima in many groups, masked heads and tails"""
    g = torch.Generator().manual_seed(27)
    V = 700001
    x = torch.randn(3, V, generator=g).to(dtype)
    x[0, ::4096] = 9.0           # 171 groups with the same maximum
    x[1, :500000] = -math.inf
    x[2, 3:] = -math.inf
    t = torch.tensor([4096, 600000, 2], dtype=torch.int32)
    lp, h, ids, tops = run_logprobs(ops, x.to(GPU), t, 64)
    wl, wh, wi, wt = S.logprobs(x, t, 64)
    assert torch.equal(ids.long(), wi)
    tol = 2.0 ** -18 * (1 + math.log(V)) ** 2
    for a, b in ((lp, wl), (h, wh), (tops, wt)):
        fine = torch.isfinite(b)
        assert torch.equal(a[~fine], b[~fine]) and bool(((a - b).abs()[fine] <= tol).all())


def test_refused_on_the_gpu(ops):
    from rust_interference_engine_amd import RieError, _lib
    import ctypes as C

    x = torch.zeros(4, 100, device=GPU)
    ent = torch.zeros(4)  # host memory
    err = C.create_string_buffer(256)
    ws = torch.empty(4096, dtype=torch.uint8, device=GPU)
    f = _lib.lib().rie_hip_k_token_logprobs
    assert f(0, x.data_ptr(), 4, 100, 100, None, None, ent.data_ptr(), 0, None, None, ws.data_ptr(), 4096, None, err, 256) == -5
    assert b"entropy is not device memory" in err.value
    assert f(0, ent.data_ptr(), 4, 1, 1, None, None, None, 0, None, None, ws.data_ptr(), 4096, None, err, 256) == -5
    with pytest.raises(RieError, match="on one GPU"):
        ops.TokenLogprobs(x, entropy=ent)
