"""The tolerances of the decoding operators' GPU tests notice what they are there for: mistakes planted in the plain form, on the CPU."""
import pytest

torch = pytest.importorskip("torch")

import decoding_exact as X  # noqa: E402
import serving_ref as S  # noqa: E402


def one_part(q, k, v, pos0, scale):
    """attention whose probabilities are rounded to f16 once, above and not below"""
    q, k, v = q.double(), k.double(), v.double()
    G = q.shape[1] // k.shape[1]
    k, v = (x.repeat_interleave(G, 1).transpose(0, 1) for x in (k, v))
    s = (q.transpose(0, 1) @ k.transpose(1, 2)) * scale
    seen = torch.arange(k.shape[1])[None] <= pos0 + torch.arange(q.shape[0])[:, None]
    s = s.masked_fill(~seen, -torch.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True)) * 64
    return ((e.half().double() @ v) / e.sum(-1, keepdim=True)).transpose(0, 1)


@pytest.mark.parametrize("new", [1, 5])
def test_a_probability_in_one_f16_part_is_noticed(new):
    from test_gpu_serving8_edges import cancelling

    b = cancelling(new, 43)
    worst = 0.0
    for i, (n, L) in enumerate(b.lens):
        r = int(b.starts[i])
        q = b.q[r:r + n]
        k, v = b.values(b.k_pages, b.k_scale, i), b.values(b.v_pages, b.v_scale, i)
        scale = b.hd ** -0.5
        o, a, size = S.attend(q, k, v, L - n, scale)
        tol = X.few_tolerance(o, a, q, k, scale, b.v_scale, L, b.dtype, size)
        wrong = one_part(q, k, v, L - n, scale)
        right = o.half().double()
        assert bool(((right - o).abs() <= tol).all())
        worst = max(worst, float(((wrong.half().double() - o).abs() / tol).max()))
    assert worst > 2, worst
