"""Pages in 8 bits on the GPU where append and attention can go wrong: values half way between two codes, scales
that are none, millions of sequences; what is rounded and what is not."""
import math
import random

import pytest

torch = pytest.importorskip("torch")

import decoding_exact as X  # noqa: E402
import serving8_ref as R8  # noqa: E402
import serving_ref as S  # noqa: E402
import test_gpu_serving8 as T8  # noqa: E402

pytestmark = pytest.mark.gpu
GPU = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "needs the MI355X"
    from rust_interference_engine_amd import ops
    return ops


def appended_like(ops, b, x, KV):
    """append to the GPU and to the plain form; both results"""
    want = []
    for codes, scale, y in ((b.k_pages, b.k_scale, x[:, :KV]), (b.v_pages, b.v_scale, x[:, KV:])):
        c, s = b.paged(codes).clone(), scale.clone()
        for i, (n, L) in enumerate(b.lens):
            r = int(b.starts[i])
            X.append(c, s, b.table[i], b.page, b.block, L - n, y[r:r + n])
        want.append((c, s))
    return T8.appended(ops, b, x[:, :KV], x[:, KV:]), [want[0][0], want[1][0], want[0][1], want[1][1]]


def test_ties_of_codes_go_to_even(ops):
    """values that lie half way between two codes, of scales whose inverse is no f64 number: 73.5 / 49 is 1.5"""
    n, hd, KV = 60, 64, 2
    b = R8.Batch8([(1, 1)] * n, KV, KV, hd, page=16, block=16, dtype=F16, seed=31)
    x = torch.zeros(n, 2 * KV, hd)
    for i in range(n):
        for h in range(2 * KV):
            s = 2 * (i * 2 * KV + h) + 3  # odd, so a half of it is a value
            x[i, h, 0] = 127 * s
            x[i, h, 1:] = (torch.arange(hd - 1) * 2 - 63 + (i % 2) * 62) / 2 * s
    x[0, 0, 0], x[0, 0, 1] = 6223, 73.5
    got, want = appended_like(ops, b, x, KV)
    T8.same(got, want)
    assert int(got[0][int(b.table[0, 0]), 0, 0, 1]) == 2


@pytest.mark.parametrize("block", [16, 64])
def test_ties_of_earlier_codes_go_to_even(ops, block):
    """a block whose scale grows from s to s': code * s / s', where that is half way; 47 * 3 / 94 is 1.5"""
    pairs = [(s, t) for s in range(1, 64) for t in range(s + 1, 200) if any((2 * c * s) % t == 0 and (2 * c * s) // t % 2 for c in range(-127, 128))]
    pairs = [(3, 94)] + random.Random(3).sample(pairs, 399)
    n, hd, KV = len(pairs) // 4, 256, 2
    b = R8.Batch8([(1, 2)] * n, KV, KV, hd, page=64, block=block, dtype=F16, seed=32)
    x = torch.zeros(n, 2 * KV, hd)
    for i in range(n):
        for h in range(2 * KV):
            s, t = pairs[4 * i + h]
            pg = int(b.table[i, 0])
            codes, scale = (b.paged(b.k_pages), b.k_scale) if h < KV else (b.paged(b.v_pages), b.v_scale)
            codes[pg, 0, h % KV, :255] = torch.arange(-127, 128, dtype=torch.int8)
            scale[pg, 0, h % KV] = s
            x[i, h, 5] = -127.0 * t
    got, want = appended_like(ops, b, x, KV)
    T8.same(got, want)
    assert int(got[0][int(b.table[0, 0]), 0, 0, 127 + 47]) == 2


def test_append_of_random_rows_to_the_bit(ops):
    b = R8.Batch8([(1, 20), (40, 90), (3, 3), (17, 33)], 2, 2, 128, page=64, block=32, dtype=F16, seed=33)
    for ty in (F32, F16, BF16):
        x = (torch.randn(b.rows, 4, 128, generator=torch.Generator().manual_seed(2)) * 40).round().to(ty)  # whole numbers: many ties
        T8.same(*appended_like(ops, b, x, 2))


@pytest.mark.parametrize("scale", [-1.0, -2.0 ** -70, 2.0 ** 51, math.inf, math.nan])
def test_scales_that_are_none_are_nan_to_append_and_attention(ops, scale):
    for lens in ([(1, 60)], [(2, 60)], [(50, 60)], [(40, 60)]):
        for which in ("k_scale", "v_scale"):
            b = R8.Batch8(lens, 8, 2, 128, page=32, block=16, dtype=BF16, seed=34)
            getattr(b, which)[b.table[0, 0].long(), 1, 0] = scale  # positions 16..31 of head 0
            out = T8.paged(ops, b)
            sees = torch.arange(lens[0][1] - lens[0][0], lens[0][1]) >= 16
            assert bool(out[sees][:, :4].isnan().all()) and not bool(out[:, 4:].isnan().any()) and not bool(out[~sees].isnan().any())
    b = R8.Batch8([(3, 20)], 2, 2, 128, page=32, block=32, dtype=F16, seed=35)
    b.k_scale[:] = b.v_scale[:] = scale
    x = torch.randn(3, 4, 128, generator=torch.Generator().manual_seed(3))
    got, want = appended_like(ops, b, x, 2)
    T8.same(got, want)
    assert bool(got[2][int(b.table[0, 0])].isnan().all())


@pytest.mark.parametrize("tiny", [2.0 ** -62, 2.0 ** -70, 2.0 ** -100])
def test_scales_that_are_too_small_count_as_the_smallest(ops, tiny):
    for lens in ([(1, 40)], [(50, 60)]):
        b = R8.Batch8(lens, 4, 2, 64, page=64, block=64, dtype=BF16, seed=36)
        b.v_scale[:] = tiny
        out = T8.paged(ops, b)
        b.v_scale[:] = X.MIN
        assert torch.equal(out, T8.paged(ops, b)) and bool((out != 0).any())
    for top in (2.0 ** -50, 2.0 ** -52, 2.0 ** -57, 0.0):
        b = R8.Batch8([(1, 20), (2, 9)], 2, 2, 64, page=32, block=32, dtype=F16, seed=37)
        b.k_scale[:] = b.v_scale[:] = tiny
        x = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(4)).clamp(-2, 2) * top
        T8.same(*appended_like(ops, b, x, 2))


def test_chunks_among_millions_of_sequences(ops):
    """more blocks of rows than workgroups of 512 threads can be launched for; all but a few sequences are empty"""
    n_seq, KV, hd, page = (1 << 23) + 5, 1, 64, 128
    some = {0: (70, 90), 1: (1, 5), 1 << 22: (3, 100), n_seq - 1: (9, 9)}
    b = R8.Batch8([some[i] for i in some], 2 * KV, KV, hd, page=page, block=64, dtype=F16, seed=51)
    at = torch.tensor(list(some))
    new, lens, table = torch.zeros(n_seq, dtype=torch.int32), torch.zeros(n_seq, dtype=torch.int32), torch.full((n_seq, 1), -1, dtype=torch.int32)
    new[at], lens[at], table[at] = torch.tensor([n for n, _ in some.values()], dtype=torch.int32), b.L, b.table[:, :1]
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), new.cumsum(0)]).int()
    kv = ops.PagedKv(b.paged(b.k_pages.to(GPU)), b.paged(b.v_pages.to(GPU)), table.to(GPU), k_scale=b.k_scale.to(GPU), v_scale=b.v_scale.to(GPU))
    out = torch.full((b.rows, 2 * KV, hd), 7.0, dtype=F16, device=GPU)
    ops.PagedAttention(kv, ops.Seqs(starts.to(GPU), lens.to(GPU), max_new=70, max_len=128), b.q.to(GPU), out)()
    T8.check(b, out.cpu())


# ---- what is rounded: of few rows the output alone ----

def check_few(b, out, window=0, softcap=0.0, scale=None):
    scale = 1 / math.sqrt(b.hd) if scale is None else scale
    for i, (n, L) in enumerate(b.lens):
        r = int(b.starts[i])
        q = b.q[r:r + n]
        k, v = b.values(b.k_pages, b.k_scale, i), b.values(b.v_pages, b.v_scale, i)
        o, a, size = S.attend(q, k, v, L - n, scale, window, softcap)
        if n:
            tol = X.few_tolerance(o, a, q, k, scale, b.v_scale, L, b.dtype, size, softcap)
            err = (out[r:r + n].double() - o).abs()
            assert bool((err <= tol).all()), (i, n, L, float((err / tol).max()))


@pytest.mark.parametrize("H,KV,hd,page,block", T8.SHAPES + [(14, 2, 64, 16, 16), (3, 1, 256, 64, 16), (32, 1, 128, 16, 16)])
@pytest.mark.parametrize("window,softcap", [(0, 0.0), (40, 0.0), (0, 5.0)])
def test_few_rows_round_their_output_only(ops, H, KV, hd, page, block, window, softcap):
    lens = [(1, 1), (1, 17), (1, 33), (1, 500), (0, 64), (1, 129)]
    b = R8.Batch8(lens, H, KV, hd, page=page, block=block, seed=41)
    check_few(b, T8.paged(ops, b, window, softcap), window, softcap)


@pytest.mark.parametrize("lens", [[(3, 300), (2, 9), (4, 40)], [(1, 5000)], [(4, 4097)], [(1, 3000), (2, 800), (1, 1700), (4, 20)], [(1, 900 + 7 * i) for i in range(66)]])
@pytest.mark.parametrize("H,KV,hd", [(8, 2, 128), (12, 4, 64), (6, 3, 96), (4, 1, 256)])
def test_few_rows_in_splits_and_pieces_round_their_output_only(ops, lens, H, KV, hd):
    b = R8.Batch8(lens, H, KV, hd, page=64, block=32, seed=42)
    check_few(b, T8.paged(ops, b))


def cancelling(new, seed):
    """two positions of nearly one weight whose values cancel: what is left is the probabilities' rounding"""
    b = R8.Batch8([(new, 64 + i) for i in range(8)], 16, 4, 128, page=64, block=64, seed=seed)
    b.q *= 0.05
    b.v_scale[:] = 1.0
    for i, (n, L) in enumerate(b.lens):
        t = b.table[i, 0].long()
        v = b.paged(b.v_pages)
        v[t, 1:64:2] = -v[t, 0:64:2]
    return b


@pytest.mark.parametrize("new", [1, 5])
def test_values_that_cancel(ops, new):
    b = cancelling(new, 43)
    check_few(b, T8.paged(ops, b))
