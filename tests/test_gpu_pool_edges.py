"""Pools of pages on the GPU where rows have been cut back into pages that other rows hold, and where they outgrow their table."""
import random

import pytest

torch = pytest.importorskip("torch")

import decoding_exact as X  # noqa: E402
import test_gpu_decoding as T  # noqa: E402

pytestmark = pytest.mark.gpu
GPU = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "needs the MI355X"
    from rust_interference_engine_amd import ops
    return ops


class Both(T.Both):
    def __init__(self, ops, rows, lens, n_pages, cols, page, seed=0, refs=None):
        super().__init__(ops, rows, lens, n_pages, cols, page, seed, refs)
        r = self.ref
        self.ref, self.seed = X.SharedPool(r.rows, r.lens, r.refs, cols, page, r.caches), seed

    def fork(self, src):
        self.ops.PageFork(self.pool, torch.tensor(src, dtype=torch.int32, device=GPU), self.bufs)()
        self.ref.fork(src)
        self.check()

    def shorten(self, lens):
        self.pool.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        self.ref.lens = list(lens)


@pytest.mark.parametrize("src", [[0, 1], [0, 0], [1, 0], [1, 1], [-1, 0], [0, 5]])
def test_a_row_cut_back_into_a_page_that_another_holds(ops, src):
    """two rows share a full page, one is cut back into it: what is written to it next has to be its own"""
    b = Both(ops, [[4, 1], [4, 2]], [20, 25], 12, 4, 16)
    b.shorten([9, 25])
    b.fork(src)
    for i, r in enumerate(b.ref.rows):
        full = b.ref.lens[i] // 16
        assert all(b.ref.refs[p] == 1 for p in r[full:])  # nobody else has what this row writes


def test_two_rows_with_one_partial_page(ops):
    b = Both(ops, [[3], [3], [3]], [5, 9, 16], 8, 2, 16)
    b.fork([0, 1, 2])
    b.fork([0, 0, 1])


def test_shared_pages_behind_the_last_position(ops):
    """pages that are held ahead and shared: not written to either, whether the length ends on a page or not"""
    for lens in ([20, 90], [16, 90], [0, 90], [40, 90], [5, 3]):
        for src in ([0, 1], [0, 0], [1, 0]):
            b = Both(ops, [[7, 1, 2, 5, 11], [7, 1, 2, 9, 10, 3]], [80, 90], 20, 7, 16)
            b.shorten(lens)
            b.fork(src)
    rows = [list(range(100)), list(range(70)) + [150, 151]]  # more pages ahead than a wave has lanes
    b = Both(ops, rows, [1600, 1152], 300, 110, 16)
    b.shorten([8, 1152])
    b.fork([0, 1])
    b = Both(ops, rows, [1600, 1152], 300, 110, 16)
    b.shorten([16 * 80 + 3, 1152])
    b.fork([0, 1])


def test_a_shared_partial_page_and_no_free_one(ops):
    b = Both(ops, [[0, 1], [0, 2]], [20, 25], 3, 4, 16)
    b.shorten([9, 25])
    b.fork([0, 1])
    assert b.pool.counts.tolist()[0] == 1 and b.pool.table[0, 0] == -1


def test_a_page_that_the_program_counts(ops):
    """a prefix's partial page that no row but one holds, and a program's own list"""
    b = Both(ops, [[2], [5]], [7, 3], 9, 3, 16, refs=[0, 0, 2, 0, 0, 1, 0, 0, 0])
    b.fork([0, 1])
    assert b.pool.refs.tolist()[2] == 1


@pytest.mark.parametrize("seed", range(8))
@pytest.mark.parametrize("n,cols,page,n_pages", [(2, 3, 16, 20), (12, 9, 16, 300), (70, 20, 4, 4000), (1500, 6, 4, 30000)])
def test_forks_between_cuts(ops, n, cols, page, n_pages, seed):
    rng = random.Random(seed * 1000 + n)
    b = Both(ops, *T.random_rows(rng, n, cols, page, n_pages, share=0.6), n_pages, cols, page, seed)
    for step in range(4):
        b.shorten([rng.choice([x, x, max(x - 1, 0), x // 2, rng.randint(0, x)]) for x in b.ref.lens])
        b.fork([rng.randrange(n) if rng.random() < 0.6 else i for i in range(n)] if step % 2 else list(range(n)))


def test_cuts_and_forks_captured_and_replayed(ops):
    rng = random.Random(9)
    n, cols, page, n_pages = 8, 6, 16, 200
    b = Both(ops, *T.random_rows(rng, n, cols, page, n_pages, share=0.7), n_pages, cols, page)
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
        b.shorten([rng.randint(0, min(x, cols * page - 1)) for x in b.ref.lens])
        src.copy_(torch.tensor(s, dtype=torch.int32))
        graph.replay()
        b.ref.fork(s)
        b.ref.lens = [x + 1 for x in b.ref.lens]
        b.ref.reserve()
        b.check()
        torch.zeros(100, device=GPU).sum().item()


def test_what_a_cut_sequence_appends_leaves_the_other_as_it_was(ops):
    """the whole use: share a prompt's pages, cut one sequence back into them, fork, reserve, append"""
    page, KV, hd, n_pages, cols = 16, 2, 64, 12, 4
    g = torch.Generator().manual_seed(1)
    pool = ops.PagePool.empty(n_pages, 2, cols, page, GPU)
    codes = torch.randint(-127, 128, (2, n_pages, KV, page, hd), generator=g, dtype=torch.int8).to(GPU)
    scales = (torch.rand(2, n_pages, 1, KV, generator=g) + 0.1).to(GPU)
    kv = ops.PagedKv(codes[0].transpose(1, 2), codes[1].transpose(1, 2), pool.table, k_scale=scales[0], v_scale=scales[1])
    pool.lens.copy_(torch.tensor([40, 0]))
    src = torch.tensor([0, 0], dtype=torch.int32, device=GPU)
    reserve, fork = ops.PageReserve(pool), ops.PageFork(pool, src, [codes[0], codes[1], scales[0], scales[1]])
    reserve(), fork()  # row 1 goes on from row 0
    held = pool.table[1, :3].long()
    before = codes[:, held].cpu(), scales[:, held].cpu()
    pool.lens[0] = 10  # row 0 is cut back into their first page
    src.copy_(torch.tensor([0, 1]))
    fork()
    x = torch.randn(30, 2 * KV, hd, generator=g).to(GPU)
    pool.lens[0] = 40
    reserve()
    assert pool.counts.tolist()[0] == 0
    seqs = ops.Seqs(torch.tensor([0, 30, 30], dtype=torch.int32, device=GPU), pool.lens, max_new=30, max_len=64)
    ops.PagedAppend(kv, seqs, x[:, :KV], x[:, KV:])()
    assert torch.equal(codes[:, held].cpu(), before[0]) and torch.equal(scales[:, held].cpu(), before[1])
    assert torch.equal(pool.table[1, :3].long(), held)


# ---- rows that outgrow their table ----

def test_reserve_counts_the_pages_that_a_table_has_no_room_for(ops):
    b = Both(ops, [[], [2], [5, 6]], [100, 200, 17], 30, 4, 16)
    reserve = ops.PageReserve(b.pool)
    reserve()
    b.ref.reserve()
    b.check()
    assert b.pool.counts.tolist()[0] == 3 + 9
    b.shorten([64, 64, 64])
    reserve()
    b.ref.reserve()
    b.check()
    assert b.pool.counts.tolist()[0] == 0
    b.shorten([2 ** 31 - 1, 2 ** 31 - 1, -5])
    reserve()
    assert b.pool.counts.tolist()[0] == 2 * (2 ** 31 // 16 - 4)


def test_reserve_counts_beyond_31_bits_as_the_largest_number(ops):
    pool = ops.PagePool.empty(9, 3000, 2, 1, GPU)
    pool.lens.fill_(2 ** 31 - 1)
    ops.PageReserve(pool)()
    assert pool.counts.tolist()[0] == 2 ** 31 - 1 and pool.held.tolist() == [2] * 4 + [1] + [0] * 2995
