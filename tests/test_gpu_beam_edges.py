"""Beam selection on the GPU at its largest sizes, and what its sums are off by."""
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


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,W,V,K", [(1, 33, 128, 128), (1, 64, 128, 128), (2, 64, 5003, 128), (1, 64, 151936, 128), (3, 40, 700, 100), (2, 64, 128, 127)])
def test_beams_whose_merge_takes_up_to_64_kilobytes(ops, n, W, V, K, dtype):
    g = torch.Generator().manual_seed(V + W)
    x = (torch.randn(n * W, V, generator=g) * 3).to(dtype)
    scores = -torch.rand(n, W, generator=g) * 2
    T.chosen(T.select(ops, x.to(GPU), scores, K), x, scores, K)


def test_the_largest_search_captured_and_replayed(ops):
    g = torch.Generator().manual_seed(5)
    x, scores = torch.randn(64, 3001, generator=g).to(GPU), -torch.rand(1, 64, generator=g).to(GPU)
    nxt, parents, tokens = (torch.empty(1, 128, dtype=t, device=GPU) for t in (F32, torch.int32, torch.int32))
    pick = ops.BeamSelect(x, scores, nxt, parents, tokens)
    pick()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pick()
    for step in range(4):
        x.copy_(torch.randn(64, 3001, generator=g))
        graph.replay()
        T.chosen((nxt.cpu(), parents.cpu(), tokens.cpu()), x, scores.cpu(), 128)
        torch.zeros(100, device=GPU).sum().item()


def sum_tolerance(x, keys, rows):
    """|error| of next_scores, of a row x (one of `rows`) in float64 with the exact sums keys.  Terms e^(x - m): the
    exponent's rounding and that of log2 e, 1.25 * 2^-24 of (m - x) in all, each with its term's weight; the exponential
    2^-23.  Additions of 2^-24: 4 in a lane's step of 1024 logits, the steps of a run (32 groups of up to 4 at most, one
    where 8192 waves are more than there are groups), 6 across lanes.  Runs are joined one behind the other by 256 threads,
    then 8 times in pairs, with a factor each (2^-22 in all).  Then one rounding to f32."""
    n = -(-x.numel() // 1024)
    steps = -(-n // 512)
    groups = -(-n // steps)
    per = min(max(-(-rows * groups // 8192), 1), 32)
    w = torch.softmax(x, -1)
    terms = float((w * (x.max() - x).nan_to_num(0.0, posinf=0.0)).sum()) * 1.25 * 2.0 ** -24
    return 2.0 ** -24 * keys.abs() + terms + (2 + 4 + steps * per + 6) * 2.0 ** -24 + (-(-groups // per) // 256 + 1 + 8) * 2.0 ** -22


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,V", [(1, 7), (4, 1000), (3, 32003), (2, 151936), (1, 600001), (70, 128256)])
@pytest.mark.parametrize("spread", [0.0, 3.0])
def test_sums_of_beams_that_are_near_zero(ops, n, V, spread, dtype):
    """scores that take the row's sum away, so that f32 shows what it is off by"""
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(n, V, generator=g) * spread + 5).to(dtype)
    lse = torch.logsumexp(x.double(), -1)
    scores = (lse - x.double().amax(-1)).float()[:, None]
    nxt, par, tok = T.select(ops, x.to(GPU), scores, 4)
    for r in range(n):
        key = scores[r, 0].double() + x[r, tok[r].long()].double() - lse[r]
        err = (nxt[r].double() - key).abs()
        tol = sum_tolerance(x[r].double(), key, n)
        assert bool((err <= tol).all()), (r, float((err / tol).max()))
        assert torch.equal(x[r, tok[r].long()].sort(descending=True).values, x[r].sort(descending=True).values[:4])
