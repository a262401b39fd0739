"""Rotary rows, beam selection's logits and pages that are copied, forked and moved beyond 2^32 bytes and elements, on the GPU."""
import pytest

torch = pytest.importorskip("torch")

import test_gpu_decoding as T  # noqa: E402

pytestmark = pytest.mark.gpu
GPU = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "needs the MI355X"
    from rust_interference_engine_amd import ops
    return ops


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_rows(ops, interleaved):
    """rows 2^30 values apart, of queries and of keys behind them; in place and to another place"""
    g = torch.Generator().manual_seed(1)
    flat = torch.zeros((1 << 32) + (1 << 12), dtype=F16, device=GPU)
    rows = flat[:(1 << 32)].view(4, 1 << 30)[:, :6 * 64].unflatten(1, (6, 64))
    x = torch.randn(4, 6, 64, generator=g).half()
    pos = torch.tensor([5, 1000, 0, 77777], dtype=torch.int32)
    f = ops.rotary_frequencies(64)[0]
    rows.copy_(x)
    out = torch.empty(4, 6, 64, dtype=F16, device=GPU)
    ops.Rotary(f.to(GPU), rows[:, :4], rows[:, 4:], out[:, :4], out[:, 4:], positions=pos.to(GPU), interleaved=interleaved)()
    T.near(out, x, pos, f, 1.0, interleaved)
    ops.Rotary(f.to(GPU), rows[:, :4], rows[:, 4:], rows[:, :4], rows[:, 4:], positions=pos.to(GPU), interleaved=interleaved)()
    assert torch.equal(rows.cpu(), out.cpu())
    ops.Rotary(f.to(GPU), out[:, :4], out[:, 4:], rows[:, 2:], rows[:, :2], positions=torch.zeros(4, dtype=torch.int32, device=GPU), interleaved=interleaved)()
    assert torch.equal(rows[:, 2:].cpu(), out[:, :4].cpu()) and torch.equal(rows[:, :2].cpu(), out[:, 4:].cpu())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_beam_logits(ops, dtype):
    g = torch.Generator().manual_seed(2)
    W, V, gap = 5, 40001, 1 << 30
    flat = torch.zeros(W * gap, dtype=dtype, device=GPU)
    x = torch.randn(W, V, generator=g).to(dtype)
    rows = flat.view(W, gap)[:, 3:3 + V]
    rows.copy_(x)
    scores = -torch.rand(1, W, generator=g)
    T.chosen(T.select(ops, rows, scores, 12), x, scores, 12)


def test_pages(ops):
    n_pages, size = 40, 1 << 27  # 5 GiB of pages, 16 values of each looked at
    cache = torch.zeros(n_pages, size, dtype=torch.uint8, device=GPU)
    at = torch.arange(0, size, size // 16, device=GPU) + 4095
    mark = torch.arange(n_pages * 16, device=GPU).view(n_pages, 16).to(torch.uint8) * 7 + 1
    cache[:, at] = mark
    ids = dict(dtype=torch.int32, device=GPU)
    src, dst = torch.tensor([39, 2], **ids), torch.tensor([1, 38], **ids)
    ops.PageCopy([cache], src, dst)()
    want = mark.clone()
    want[1], want[38] = mark[39], mark[2]
    assert torch.equal(cache[:, at], want)
    pool = ops.PagePool.empty(n_pages, 2, 3, 16, GPU)
    pool.table[0, :2] = torch.tensor([36, 37], **ids)
    pool.lens[0], pool.held[0] = 20, 2
    pool.refs[36] = pool.refs[37] = 1
    pool.refs[:34] = 1  # a program's own: the copy goes to page 34
    ops.PageFork(pool, torch.zeros(2, **ids), [cache])()
    want[34] = want[37]
    assert torch.equal(cache[:, at], want) and pool.table[:, :2].tolist() == [[36, 37], [36, 34]]
    pool.refs[:34] = 0
    ops.PageCompact(pool, [cache])()
    want[0], want[1], want[2] = want[34].clone(), want[36].clone(), want[37].clone()
    assert torch.equal(cache[:, at], want) and pool.table[:, :2].tolist() == [[1, 2], [1, 0]]
