"""The paged cache in 8 bits on the GPU against plain float64 forms: what append writes, to the bit, and attention over it;
sizes, masks and layouts where they can go wrong."""
import math

import pytest

torch = pytest.importorskip("torch")

import serving8_ref as R  # noqa: E402
import serving_ref as S  # noqa: E402

pytestmark = pytest.mark.gpu
GPU = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
SHAPES = [(4, 1, 32, 16, 16), (15, 5, 64, 32, 16), (6, 3, 96, 16, 16), (8, 2, 128, 128, 64), (8, 1, 128, 16, 16), (4, 1, 256, 32, 32), (7, 7, 128, 64, 32)]


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "needs the MI355X"
    from rust_interference_engine_amd import ops
    return ops


def paged(ops, b, window=0, softcap=0.0, scale=None, max_new=None, max_len=None, fill=7.0):
    """outputs of the paged call on the CPU; rows outside the sequences keep `fill`"""
    kv = ops.PagedKv(b.paged(b.k_pages.to(GPU)), b.paged(b.v_pages.to(GPU)), b.table.to(GPU), k_scale=b.k_scale.to(GPU), v_scale=b.v_scale.to(GPU))
    seqs = ops.Seqs(b.starts.to(GPU), b.L.to(GPU), max_new=max_new or b.max_new(), max_len=max_len or b.max_len())
    out = torch.full((b.rows, b.H, b.hd), fill, dtype=b.dtype, device=GPU)
    call = ops.PagedAttention(kv, seqs, b.q.to(GPU), out, scale=scale, window=window, softcap=softcap)
    call()
    first = out.cpu()
    call()
    again = bool((out.cpu().nan_to_num(5.0) == first.nan_to_num(5.0)).all())
    assert again, "other bits the second time"
    return first


def check(b, out, window=0, softcap=0.0, scale=None, fill=7.0):
    scale = 1 / math.sqrt(b.hd) if scale is None else scale
    for i, (n, L) in enumerate(b.lens):
        r = int(b.starts[i])
        q = b.q[r:r + n]
        k, v = b.values(b.k_pages, b.k_scale, i), b.values(b.v_pages, b.v_scale, i)
        o, a, size = S.attend(q, k, v, L - n, scale, window, softcap)
        tol = R.tolerance(o, a, q, k, v, scale, L, b.hd, b.dtype, size, softcap)
        err = (out[r:r + n].double() - o).abs()
        assert bool((err <= tol).all()), (i, n, L, float((err / tol).max()))
    assert bool((out[int(b.starts[-1]):] == fill).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,KV,hd,page,block", SHAPES + [(14, 2, 64, 16, 16), (3, 1, 256, 64, 16)])
def test_single_tokens(ops, H, KV, hd, page, block, dtype):
    b = R.Batch8([(1, 1), (1, 17), (1, 32), (1, 33), (1, 0), (1, 500), (0, 64), (1, 129)], H, KV, hd, page=page, block=block, dtype=dtype, extra_rows=2, extra_cols=1)
    check(b, paged(ops, b))


@pytest.mark.parametrize("page,block", [(16, 16), (64, 16), (64, 64), (256, 128)])
@pytest.mark.parametrize("H,KV,hd", [(8, 2, 128), (4, 1, 256), (8, 8, 64)])
@pytest.mark.parametrize("window,softcap", [(0, 0.0), (40, 0.0), (0, 5.0), (1, 2.0)])
def test_a_few_tokens_of_each_sequence(ops, H, KV, hd, page, block, window, softcap):
    b = R.Batch8([(3, 3), (2, 100), (4, 515), (1, 40), (3, 2), (4, 4)], H, KV, hd, page=page, block=block, dtype=BF16, seed=1)
    check(b, paged(ops, b, window, softcap), window, softcap)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,KV,hd,page,block", SHAPES)
@pytest.mark.parametrize("window,softcap", [(0, 0.0), (70, 0.0), (0, 3.0)])
def test_chunks_and_single_tokens_in_one_batch(ops, H, KV, hd, page, block, dtype, window, softcap):
    b = R.Batch8([(1, 300), (37, 37), (65, 400), (0, 9), (1, 1), (130, 131), (5, 2)], H, KV, hd, page=page, block=block, dtype=dtype, seed=2, extra_rows=3)
    check(b, paged(ops, b, window, softcap), window, softcap)


@pytest.mark.parametrize("lens", [[(1, 5000)], [(2, 4097), (1, 3)], [(40, 6000)], [(1, 4096)] * 3])
@pytest.mark.parametrize("hd", [64, 128])
def test_long_caches_in_splits(ops, lens, hd):
    b = R.Batch8(lens, 8, 2, hd, page=64, block=32, dtype=F16, seed=3)
    check(b, paged(ops, b))
    check(b, paged(ops, b, 1500), 1500)
    check(b, paged(ops, b, max_len=6000))


@pytest.mark.parametrize("lens", [[(1, 33), (3, 90)], [(9, 90), (40, 70)]])  # few rows; tiles
def test_rows_of_pages_in_either_order_and_a_scale(ops, lens):
    b = R.Batch8(lens, 8, 4, 64, page=32, seed=4, order="slots")
    check(b, paged(ops, b, scale=0.31), scale=0.31)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("G,new", [(16, 1), (17, 1), (4, 5), (8, 4), (32, 1), (33, 1)])
@pytest.mark.parametrize("window", [0, 40])
def test_sixteen_to_thirty_three_rows_of_a_sequence(ops, G, new, hd, window, dtype):
    b = R.Batch8([(new, 100), (1, 60), (new, new)], 2 * G, 2, hd, page=32, dtype=dtype, seed=5)
    check(b, paged(ops, b, window), window)


@pytest.mark.parametrize("lens", [[(1, 700), (3, 900)], [(60, 700), (1, 800)]])
def test_scales_that_differ_by_far(ops, lens):
    """of keys, so that the maximum moves; of values, 2^-20 to 2^20 of one another: what counts are the large ones"""
    b = R.Batch8(lens, 4, 2, 64, page=32, seed=6, dtype=BF16)
    g = torch.Generator().manual_seed(1)
    b.k_scale *= 10 ** (torch.rand(b.k_scale.shape, generator=g) * 1.5 - 0.5)
    b.v_scale *= 2.0 ** torch.randint(-20, 21, b.v_scale.shape, generator=g)
    check(b, paged(ops, b))


@pytest.mark.parametrize("lens", [[(1, 700), (3, 90)], [(60, 700), (1, 90)]])
@pytest.mark.parametrize("power", [-45, 40])
def test_values_of_any_size(ops, lens, power):
    b = R.Batch8(lens, 4, 2, 128, page=32, seed=7, dtype=BF16)
    b.v_scale *= 2.0 ** power
    b.k_scale *= 2.0 ** -power
    b.q = (b.q.float() * 2.0 ** power).to(BF16)
    check(b, paged(ops, b))


@pytest.mark.parametrize("lens", [[(1, 700), (3, 90)], [(60, 700), (1, 90)]])
def test_blocks_of_zeros(ops, lens):
    """as append leaves them: codes and scales of zero; a block that alone is seen among them"""
    b = R.Batch8(lens, 4, 2, 128, page=16, seed=8)
    for s, c in ((b.k_scale, b.k_pages), (b.v_scale, b.v_pages)):
        z = torch.rand(s.shape, generator=torch.Generator().manual_seed(2)) < 0.4
        z[b.table[1, 0].long(), 0] = True
        s[z] = 0
        c[z[:, 0]] = 0  # one block to a page; heads first
    check(b, paged(ops, b))


@pytest.mark.parametrize("window", [0, 20])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("H,KV,hd,new", [(8, 2, 128, 60), (8, 2, 64, 3), (4, 1, 256, 40), (4, 2, 32, 2), (12, 2, 96, 2), (12, 2, 96, 70)])
def test_a_nan_scale_spoils_the_tokens_that_see_its_block(ops, H, KV, hd, new, which, window):
    L = 200
    b = R.Batch8([(new, L), (1, 70)], H, KV, hd, page=32, block=16, dtype=BF16, seed=9)
    clean = paged(ops, b, window)
    for at in (L - 2, L - 40, 3):
        keep = getattr(b, which + "_scale").clone()
        getattr(b, which + "_scale")[int(b.table[0, at // 32]), at % 32 // 16, 0] = math.nan
        out = paged(ops, b, window)
        getattr(b, which + "_scale").copy_(keep)
        pos = torch.arange(L - new, L)
        b0 = at // 16 * 16
        hit = pos >= b0
        if window:
            hit &= pos - window + 1 <= b0 + 15
        G = H // KV
        others = bool((out[new:] == clean[new:]).all()), bool((out[:new, G:] == clean[:new, G:]).all()), bool((out[:new, :G][~hit] == clean[:new, :G][~hit]).all())
        assert all(others) and bool(out[:new, :G][hit].isnan().all()), others


@pytest.mark.parametrize("new", [1, 50])
def test_positions_of_pages_that_are_none_are_not_seen(ops, new):
    b = R.Batch8([(new, 200), (1, 40)], 8, 2, 128, page=32, seed=10)
    b.table[0, 2], b.table[0, 4], b.table[1, :] = -3, b.n_pages, 2 ** 31 - 1
    out = paged(ops, b)
    assert bool((out[new:] == 0).all())
    k, v = (torch.cat([b.values(c, s, 0, 64), torch.zeros(136, 2, 128)]) for c, s in ((b.k_pages, b.k_scale), (b.v_pages, b.v_scale)))
    seen = torch.ones(200, dtype=torch.bool)
    seen[64:96] = seen[128:160] = False
    t = b.table[0].clone()
    t[2] = t[4] = 0
    b.table[0] = t
    k, v = b.values(b.k_pages, b.k_scale, 0)[seen], b.values(b.v_pages, b.v_scale, 0)[seen]
    pos = torch.arange(200)[seen]
    for i in range(new):
        n = int((pos <= 200 - new + i).sum())
        o, a, size = S.attend(b.q[i:i + 1], k[:n], v[:n], n - 1, 128 ** -0.5)
        tol = R.tolerance(o, a, b.q[i:i + 1], k, v, 128 ** -0.5, n, 128, F16, size)
        assert bool(((out[i:i + 1].double() - o).abs() <= tol).all())


@pytest.mark.parametrize("more", [[], [(70, 52), (30, 49), (20, 90)]])  # with the chunks, the tile kernel
@pytest.mark.parametrize("window", [0, 1, 40])
def test_tokens_past_the_table_see_what_it_addresses(ops, more, window):
    b = R.Batch8([(2, 48), (3, 40), (1, 33)] + more, 4, 2, 64, page=16, seed=11)
    cap = 32
    b.table = b.table[:, :2].contiguous()
    out = paged(ops, b, window, max_len=4000)
    for i, (n, L) in enumerate(b.lens):
        r = int(b.starts[i])
        k, v = (b.values(c, s, i, min(L, cap)) for c, s in ((b.k_pages, b.k_scale), (b.v_pages, b.v_scale)))
        q = b.q[r:r + n]
        o, a, size = S.attend(q, k, v, L - n, 1 / 8, window)
        tol = R.tolerance(o, a, q, k, v, 1 / 8, L, 64, F16, size)
        assert bool(((out[r:r + n].double() - o).abs() <= tol).all()), i


@pytest.mark.parametrize("new", [2, 50])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_query_that_is_nan_or_infinite_spoils_its_own_row_only(ops, new, dtype):
    b = R.Batch8([(new, 100), (1, 30)], 8, 2, 128, seed=12, dtype=dtype)
    clean = paged(ops, b)
    b.q[1, 3, 5], b.q[0, 6, 7] = math.nan, math.inf
    out = paged(ops, b)
    hit = torch.zeros(out.shape[:2], dtype=torch.bool)
    hit[1, 3] = hit[0, 6] = True
    assert torch.equal(out[~hit], clean[~hit]) and bool(out[hit].isnan().all())


def test_slots_behind_the_last_position_may_hold_anything(ops):
    b = R.Batch8([(1, 20), (30, 40)], 8, 2, 128, page=64, block=16, seed=13)
    clean = paged(ops, b)
    for i, L in ((0, 32), (1, 48)):  # blocks that hold no position
        b.k_scale[int(b.table[i, 0]), L // 16:] = math.nan
        b.v_scale[int(b.table[i, 0]), L // 16:] = math.nan
    assert torch.equal(paged(ops, b), clean)


# ---- append ----

def appended(ops, b, k, v):
    """codes and scales after the call, on the CPU; [pages, page, KV, hd]"""
    kp, vp, ks, vs = (x.to(GPU) for x in (b.k_pages, b.v_pages, b.k_scale, b.v_scale))
    kv = ops.PagedKv(b.paged(kp), b.paged(vp), b.table.to(GPU), k_scale=ks, v_scale=vs)
    ops.PagedAppend(kv, ops.Seqs(b.starts.to(GPU), b.L.to(GPU), max_new=b.max_new(), max_len=b.max_len()), k.to(GPU), v.to(GPU))()
    return [x.cpu() for x in (b.paged(kp), b.paged(vp), ks, vs)]


def wanted(b, k, v):
    got = []
    for codes, scale, x in ((b.k_pages, b.k_scale, k), (b.v_pages, b.v_scale, v)):
        c, s = b.paged(codes).clone(), scale.clone()
        for i, (n, L) in enumerate(b.lens):
            r, first = int(b.starts[i]), L - n
            skip, cap = max(0, -first), b.table.shape[1] * b.page
            y = x[r + skip:r + max(skip, min(n, cap - first))]
            if y.shape[0]:
                R.append(c, s, b.table[i], b.page, b.block, first + skip, y)
        got.append((c, s))
    return got[0][0], got[1][0], got[0][1], got[1][1]


def same(got, want):
    for x, y in zip(got, want):
        assert torch.equal(x.nan_to_num(-9.0) if x.is_floating_point() else x, y.nan_to_num(-9.0) if y.is_floating_point() else y)


@pytest.mark.parametrize("src", [F32, F16, BF16])
@pytest.mark.parametrize("hd,page,block", [(32, 16, 16), (64, 64, 32), (96, 32, 16), (128, 128, 128), (256, 16, 16), (256, 64, 64)])
@pytest.mark.parametrize("order", ["heads", "slots"])
def test_append(ops, src, hd, page, block, order):
    b = R.Batch8([(1, 1), (1, 20), (40, 40), (0, 9), (5, 3), (100, 333), (1, 16), (1, 17), (16, 48), (130, 150)], 6, 3, hd, page=page, block=block, seed=14,
                 extra_rows=2, order=order)
    g = torch.Generator().manual_seed(3)
    x = torch.randn(b.rows, 6, hd, generator=g).to(src)  # keys and values of a token in one row
    x[::7] *= 3
    same(appended(ops, b, x[:, :3], x[:, 3:]), wanted(b, x[:, :3], x[:, 3:]))


def test_append_of_one_token_after_another(ops):
    """40 steps of one sequence: scales that grow, codes that follow"""
    b = R.Batch8([(1, 40)], 2, 2, 64, page=32, block=32, seed=15)
    b.k_scale.fill_(math.nan)  # pages that nobody has written yet
    b.v_scale.fill_(math.nan)
    g = torch.Generator().manual_seed(4)
    x = (torch.randn(40, 4, 64, generator=g) * torch.linspace(0.2, 3, 40)[:, None, None]).to(BF16)
    kp, vp, ks, vs = (y.to(GPU) for y in (b.k_pages, b.v_pages, b.k_scale, b.v_scale))
    kv = ops.PagedKv(b.paged(kp), b.paged(vp), b.table.to(GPU), k_scale=ks, v_scale=vs)
    lens, row = torch.zeros(1, dtype=torch.int32, device=GPU), torch.empty(1, 4, 64, dtype=BF16, device=GPU)
    call = ops.PagedAppend(kv, ops.Seqs(torch.tensor([0, 1], dtype=torch.int32, device=GPU), lens, max_new=1, max_len=64), row[:, :2], row[:, 2:])
    ck, cv, sk, sv = b.paged(b.k_pages).clone(), b.paged(b.v_pages).clone(), b.k_scale.clone(), b.v_scale.clone()
    for i in range(40):
        lens.fill_(i + 1)
        row.copy_(x[i:i + 1])
        call()
        R.append(ck, sk, b.table[0], 32, 32, i, x[i:i + 1, :2])
        R.append(cv, sv, b.table[0], 32, 32, i, x[i:i + 1, 2:])
    same([y.cpu() for y in (b.paged(kp), b.paged(vp), ks, vs)], [ck, cv, sk, sv])
    t = b.table[0, :2].long()
    near = (ck[t].double() * sk[t].double().repeat_interleave(32, 1)[..., None]).reshape(-1, 2, 64)[:40]
    step = sk[t].double().repeat_interleave(32, 1)[..., None].reshape(-1, 2, 1)[:40]
    assert float(((near - x[:, :2].double()).abs() / step).max()) < 5  # half a step each time a scale grew


@pytest.mark.parametrize("odd", [math.nan, math.inf, 2.0 ** 58, 2.0 ** -48, 2.0 ** -55, 0.0])
@pytest.mark.parametrize("n,L", [(1, 8), (5, 30), (40, 70)])
def test_append_of_odd_values(ops, odd, n, L):
    b = R.Batch8([(n, L), (2, 9)], 2, 2, 128, page=32, block=16, seed=16)
    x = torch.randn(n + 2, 4, 128, generator=torch.Generator().manual_seed(5))
    if odd < 1:
        x[:n, 1] = odd
        b.k_scale[:] = 0.0
        b.paged(b.k_pages)[:] = 0
    else:
        x[n // 2, 1, 9] = odd
    got = appended(ops, b, x[:, :2], x[:, 2:])
    same(got, wanted(b, x[:, :2], x[:, 2:]))


def test_append_to_a_block_that_is_spoiled(ops):
    """a NaN scale stays until the block's first position comes again"""
    b = R.Batch8([(1, 8), (1, 17), (20, 25), (3, 33)], 2, 2, 64, page=64, block=16, seed=17)
    b.k_scale[:] = math.nan
    b.v_scale[:] = -1.0  # no scale either
    x = torch.randn(25, 4, 64, generator=torch.Generator().manual_seed(6))
    got = appended(ops, b, x[:, :2], x[:, 2:])
    same(got, wanted(b, x[:, :2], x[:, 2:]))
    t = b.table[:, 0].long()
    assert bool(got[2][t[0], 0].isnan().all()) and bool(torch.isfinite(got[2][t[1], 1]).all()) and bool(torch.isfinite(got[2][t[2], 1]).all())


def test_append_rounds_to_nearest_even(ops):
    b = R.Batch8([(1, 1)], 1, 1, 32, seed=18)
    x = torch.zeros(1, 2, 32)
    x[0, 0, :8] = torch.tensor([127.0, 0.5, 1.5, -0.5, -2.5, 3.4999999, 100.5, -127.0])  # a scale of one
    got = appended(ops, b, x[:, :1], x[:, 1:])
    assert got[0][int(b.table[0, 0]), 0, 0, :8].tolist() == [127, 0, 2, 0, -2, 4, 100, -127]  # 3.4999999 is 3.5 in f32
    assert float(got[2][int(b.table[0, 0]), 0, 0]) == 1.0 and float(got[3][int(b.table[0, 0]), 0, 0]) == 0.0


@pytest.mark.parametrize("new", [1, 30])
def test_append_leaves_pages_that_are_none_alone(ops, new):
    b = R.Batch8([(new, 64), (new, new)], 4, 2, 64, page=16, seed=19)
    b.table[0, -1], b.table[1, 0] = b.n_pages, -1
    x = torch.randn(2 * new, 4, 64, generator=torch.Generator().manual_seed(7))
    same(appended(ops, b, x[:, :2], x[:, 2:]), wanted(b, x[:, :2], x[:, 2:]))


def test_append_drops_the_tokens_past_the_table(ops):
    b = R.Batch8([(20, 48), (1, 40), (40, 40)], 4, 2, 64, page=16, seed=20)
    b.table = b.table[:, :2].contiguous()
    x = torch.randn(b.rows, 4, 64, generator=torch.Generator().manual_seed(8))
    same(appended(ops, b, x[:, :2], x[:, 2:]), wanted(b, x[:, :2], x[:, 2:]))


@pytest.mark.parametrize("n_seq", [63, 64, 200, 2100])
def test_many_sequences(ops, n_seq):
    lens = [(1 + i % 2, 1 + i * 7 % 90) for i in range(n_seq)]
    lens = [(min(n, x), x) for n, x in lens]
    b = R.Batch8(lens, 4, 2, 32, page=32, seed=21)
    check(b, paged(ops, b))
    x = torch.randn(b.rows, 4, 32, generator=torch.Generator().manual_seed(9))
    same(appended(ops, b, x[:, :2], x[:, 2:]), wanted(b, x[:, :2], x[:, 2:]))


def test_a_step_captured_and_replayed(ops):
    """append and attention in one graph, replayed as sequences grow, with eager work between; every replay checked"""
    b = R.Batch8([(1, 30), (1, 47), (1, 200)], 8, 2, 64, page=16, seed=22, extra_cols=3)
    t = torch.arange(b.table.numel(), dtype=torch.int32).view(b.table.shape)  # room to grow: pages for every entry
    n = b.table.numel()
    g = torch.Generator().manual_seed(10)
    codes = [torch.randint(-127, 128, (n, 2, 16, 64), generator=g, dtype=torch.int8) for _ in range(2)]
    scale = [torch.rand(n, 1, 2, generator=g) * 0.03 + 0.01 for _ in range(2)]
    dev = [x.to(GPU) for x in codes + scale]
    b.table, b.k_pages, b.v_pages, b.k_scale, b.v_scale, b.n_pages = t, codes[0], codes[1], scale[0], scale[1], n
    kv = ops.PagedKv(b.paged(dev[0]), b.paged(dev[1]), t.to(GPU), k_scale=dev[2], v_scale=dev[3])
    lens, x, q = b.L.to(GPU), torch.empty(3, 4, 64, device=GPU), torch.empty(3, 8, 64, dtype=F16, device=GPU)
    out = torch.zeros(3, 8, 64, dtype=F16, device=GPU)
    seqs = ops.Seqs(b.starts.to(GPU), lens, max_new=1, max_len=240)
    append, attend = ops.PagedAppend(kv, seqs, x[:, :2], x[:, 2:]), ops.PagedAttention(kv, seqs, q, out)
    graph = torch.cuda.CUDAGraph()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        append(), attend()
    torch.cuda.synchronize()
    for d, h in zip(dev, codes + scale):
        d.copy_(h)
    with torch.cuda.graph(graph):
        append(), attend()
    for step in range(6):
        new = torch.randn(3, 4, 64, generator=g)
        b.q = torch.randn(3, 8, 64, generator=g).half()
        b.lens = [(1, x + 1) for _, x in b.lens]
        x.copy_(new), q.copy_(b.q)
        lens += 1
        graph.replay()
        got = out.cpu()
        want = wanted(b, new[:, :2], new[:, 2:])
        same([b.paged(dev[0]).cpu(), b.paged(dev[1]).cpu(), dev[2].cpu(), dev[3].cpu()], want)
        b.paged(b.k_pages).copy_(want[0]), b.paged(b.v_pages).copy_(want[1])
        b.k_scale, b.v_scale = want[2], want[3]
        check(b, got)
        torch.zeros(1000, device=GPU).sum().item()


def test_two_calls_at_once_on_two_streams(ops):
    b = R.Batch8([(1, 9000)], 8, 2, 128, page=64, seed=23)
    kv = ops.PagedKv(b.paged(b.k_pages.to(GPU)), b.paged(b.v_pages.to(GPU)), b.table.to(GPU), k_scale=b.k_scale.to(GPU), v_scale=b.v_scale.to(GPU))
    seqs = ops.Seqs(b.starts.to(GPU), b.L.to(GPU), max_new=1, max_len=9000)
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


@pytest.mark.parametrize("new", [1, 40])
def test_offsets_past_four_gigabytes(ops, new):
    """pages whose codes lie beyond 2^32 bytes"""
    n_pages, KV, hd, page = 2 ** 15 + 40, 8, 128, 128
    codes = torch.zeros(n_pages, KV, page, hd, dtype=torch.int8, device=GPU)
    scales = [torch.ones(n_pages, 1, KV, device=GPU) * 0.01 for _ in range(2)]
    last = torch.tensor([[n_pages - 1, n_pages - 2]], dtype=torch.int32)
    b = R.Batch8([(new, 200)], KV, KV, hd, page=page, block=128, seed=24)
    kv = ops.PagedKv(codes.transpose(1, 2), codes.transpose(1, 2), last.to(GPU), k_scale=scales[0], v_scale=scales[1])
    seqs = ops.Seqs(b.starts.to(GPU), b.L.to(GPU), max_new=new, max_len=200)
    fill = torch.randint(-127, 128, (2, KV, page, hd), generator=torch.Generator().manual_seed(11), dtype=torch.int8)
    codes[last[0].long()] = fill.to(GPU)
    out = torch.empty(new, KV, hd, dtype=F16, device=GPU)
    ops.PagedAttention(kv, seqs, b.q.to(GPU), out)()
    x = (fill.transpose(1, 2).reshape(-1, KV, hd)[:200]).double() * torch.tensor(0.01).double()
    o, a, size = S.attend(b.q, x, x, 200 - new, hd ** -0.5)
    tol = R.tolerance(o, a, b.q, x, x, hd ** -0.5, 200, hd, F16, size)
    assert bool(((out.cpu().double() - o).abs() <= tol).all())


def test_refused_on_the_gpu(ops):
    from rust_interference_engine_amd import RieError
    b = R.Batch8([(1, 30)], 4, 2, 64, page=32)
    k, v, t, ks, vs = (x.to(GPU) for x in (b.paged(b.k_pages), b.paged(b.v_pages), b.table, b.k_scale, b.v_scale))
    seqs = ops.Seqs(b.starts.to(GPU), b.L.to(GPU), max_new=1, max_len=30)
    kv = ops.PagedKv(k, v, t, k_scale=ks, v_scale=vs)
    q = b.q.to(GPU)

    def refused(text, f):
        with pytest.raises(RieError, match=text):
            f()

    refused("k_scale and v_scale", lambda: ops.PagedKv(k, v, t))
    refused("k_scale and v_scale", lambda: ops.PagedKv(k, v, t, k_scale=ks))
    refused("k_scale and v_scale", lambda: ops.PagedKv(k.half(), v.half(), t, k_scale=ks, v_scale=vs))
    refused("f32 is wanted", lambda: ops.PagedKv(k, v, t, k_scale=ks.half(), v_scale=vs.half()))
    refused("scales have to be", lambda: ops.PagedKv(k, v, t, k_scale=ks[:-1], v_scale=vs[:-1]))
    refused("scales have to be", lambda: ops.PagedKv(k, v, t, k_scale=ks[:, :, 0], v_scale=vs[:, :, 0]))
    refused("one GPU", lambda: ops.PagedKv(k, v, t, k_scale=ks.cpu(), v_scale=vs.cpu()))
    refused("block has to be", lambda: ops.PagedAttention(ops.PagedKv(k, v, t, k_scale=ks.repeat(1, 2, 1), v_scale=vs.repeat(1, 2, 1)), seqs, q, torch.empty_like(q))())
    refused("overlap", lambda: ops.PagedAppend(ops.PagedKv(k, v, t, k_scale=ks[:, :1].expand(-1, 2, -1), v_scale=vs[:, :1].expand(-1, 2, -1)), seqs, q[:, :2], q[:, 2:]))
    refused("overlap", lambda: ops.PagedAppend(ops.PagedKv(k, v, t, k_scale=ks, v_scale=ks), seqs, q[:, :2], q[:, 2:])())
    refused("f16 or bf16", lambda: ops.PagedAttention(kv, seqs, q.float(), torch.empty_like(q, dtype=F32))())
    refused("heads", lambda: ops.PagedAppend(kv, seqs, q, q))
