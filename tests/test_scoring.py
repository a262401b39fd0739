"""Scoring over the Backend boundary: Engine.score and Engine.perplexity (engine.rs:567-602) over the oracle on the CPU,
and HipBackend.forward_logprobs, which forms log probabilities on the device, on the GPU against the float64 ones of the
same backend's logits."""
import math

import numpy as np
import pytest

import rust_interference_engine_amd as R
from rust_interference_engine_amd import synth
from ggml_np import F16

TOKS = [1] + [3 + (i * 11) % 200 for i in range(29)]


def _log_softmax(x):
    x = np.asarray(x, np.float64)
    x = x - x.max(-1, keepdims=True)
    return x - np.log(np.exp(x).sum(-1, keepdims=True))


def _tol(x):
    """of the device's f32 numbers: logits within R of each other round in a handful of steps of 2^-24 R and of ln V; the
    exponentials are off by 2^-22 + R 2^-23, their sum of V by (V / 64 + 40) 2^-24"""
    r, v = float(x.max() - x.min()), x.shape[-1]
    return 3 * (r + math.log(v) + 1) * 2.0 ** -24 + (v / 64 + 40) * 2.0 ** -24 + 2.0 ** -21 + r * 2.0 ** -22


def test_score_and_perplexity_over_the_oracle(oracle):
    g = synth.build(synth.tiny("llama", F16))
    m = oracle.Model(g)
    e = R.Engine(oracle.Backend(m, 32, 8, n_threads=2))
    lp = e.score(TOKS)
    one = oracle.Backend(m, 32, 8, n_threads=2)
    want = [_log_softmax(one.forward([t], i))[TOKS[i + 1]] for i, t in enumerate(TOKS[:-1])]
    assert lp.shape == (29,) and np.abs(lp - want).max() < 1e-4 and e.cached == TOKS[:-1]
    assert abs(e.perplexity(TOKS) / math.exp(-np.mean(want)) - 1) < 1e-4
    long = TOKS + TOKS[1:9]  # 38 tokens in windows of 32
    both = np.concatenate([e.score(long[:32]), e.score(long[32:])])
    assert abs(e.perplexity(long) - math.exp(-both.mean())) < 1e-9
    assert e.score(TOKS[:1]).size == 0
    with pytest.raises(R.RieError, match="exceeds context window"):
        e.score([1] * 33)
    with pytest.raises(R.RieError, match="two tokens"):
        e.perplexity([1])


@pytest.mark.parametrize("bad", [-1, 1 << 30, 1 << 40])
def test_score_refuses_a_last_token_that_is_none(oracle, bad):
    e = R.Engine(oracle.Backend(oracle.Model(synth.build(synth.tiny("llama", F16))), 32, 8, n_threads=2))
    e.eval_tokens(TOKS[:3])
    for call in (e.score, e.perplexity):
        with pytest.raises(R.RieError, match="out of range"):
            call(TOKS[:4] + [bad])
    assert e.cached == TOKS[:3]  # refused before anything was evaluated


@pytest.mark.gpu
@pytest.mark.parametrize("arch", ["llama", "qwen3", "gemma2", "qwen3moe"])
def test_forward_logprobs_are_those_of_the_logits(arch):
    g = synth.build(synth.tiny(arch, F16))
    be, plain = R.HipBackend(g, n_ctx=64, max_batch=8), R.HipBackend(g, n_ctx=64, max_batch=8)
    V = be.n_vocab
    pos = 0
    for n, top, with_targets in ((8, 5, True), (1, 20, True), (3, 0, True), (8, 64, False), (1, 0, True), (1, 1, True)):
        toks = [(7 * (pos + i) + 3) % V for i in range(n)]
        want = [(5 * (pos + i)) % V for i in range(n)]
        if n > 2:
            want[1] = 0xFFFFFFFF  # no token
        lp, h, ids, tops = be.forward_logprobs(toks, pos, want if with_targets else None, top)
        x = plain.forward(toks, pos, True).reshape(n, V)
        p, tol = _log_softmax(x), _tol(x)
        assert np.abs(h - -(np.exp(p) * p).sum(1)).max() <= tol * (1 + 2 * math.log(V))
        order = np.argsort(-x, axis=1, kind="stable")[:, :top]
        assert ids.shape == (n, top) and (ids == order).all()
        assert not top or np.abs(tops - np.take_along_axis(p, order, 1)).max() <= tol
        assert (lp is None) == (not with_targets)
        for i in range(n if with_targets else 0):
            assert math.isnan(lp[i]) if want[i] >= V else abs(lp[i] - p[i, want[i]]) <= tol
        assert np.array_equal(be.hidden(), plain.hidden())
        pos += n


@pytest.mark.gpu
def test_forward_logprobs_refuses_and_leaves_the_backend_as_it_was():
    g = synth.build(synth.tiny("llama", F16))
    be = R.HipBackend(g, n_ctx=16, max_batch=4)
    be.forward([1, 2, 3], 0)
    for args, text in ((([], 3), "empty batch"), (([1] * 5, 3), "exceeds max batch"), (([1], 16), "context window full"), (([be.n_vocab], 3), "out of range"),
                       (([1, 2], 3, [1]), "targets for"), (([1], 3, None, 65), "n_top"), (([1], 3, None, -1), "n_top")):
        with pytest.raises(R.RieError, match=text):
            be.forward_logprobs(*args)
    assert R._lib.lib().rie_hip_forward_logprobs(be._h, None, 1, 3, None, 0, None, None, None, None, None, 0) == -5
    a = be.forward([4], 3)
    fresh = R.HipBackend(g, n_ctx=16, max_batch=4)
    fresh.forward([1, 2, 3], 0)
    assert np.array_equal(a, fresh.forward([4], 3))


@pytest.mark.gpu
def test_engine_scores_on_the_device_as_on_the_host():
    g = synth.build(synth.tiny("llama", F16))
    be = R.HipBackend(g, n_ctx=32, max_batch=8)
    e = R.Engine(be)
    lp = e.score(TOKS)
    ref = R.HipBackend(g, n_ctx=32, max_batch=8)
    want, tol = [], 0.0
    for pos in range(0, 29, 8):
        n = min(8, 29 - pos)
        x = ref.forward(TOKS[pos:pos + n], pos, True).reshape(n, -1)
        tol = max(tol, _tol(x))
        want += [_log_softmax(r)[TOKS[pos + i + 1]] for i, r in enumerate(x)]
    assert np.abs(lp - want).max() <= tol
    assert abs(e.perplexity(TOKS) / math.exp(-np.mean(want)) - 1) <= 2 * tol
    # the cache holds the text: generation goes on from it
    nxt = be.forward_argmax([TOKS[-1]], 29)
    assert nxt == int(np.argmax(ref.forward([TOKS[-1]], 29)))
