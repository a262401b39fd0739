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
