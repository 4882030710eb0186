"""route_topk on the GPU against its definition in 64 bits: scores, biases,
groups, ties, masked experts, odd counts of experts."""
import numpy as np
import pytest

import herbert_hip as hb
from route_ref import route
from test_gpu_f8 import Bufs

pytestmark = pytest.mark.gpu

# A weight: an exponential and a sigmoid of few ulp, at most 32 additions, a
# division and a product.
REL = 48 * 2.0 ** -24


def run(gpu, s, bias=None, odd=0, **kw):
    m, e = s.shape
    k = kw["top_k"]
    desc = hb.route_topk(e, bias=bias is not None, f32=s.dtype == np.float32, **kw)
    with Bufs(gpu) as b:
        r = [b.put(s, odd), b.put(np.full((m, 2 * k), 0xEE, np.uint32))] + ([b.put(bias)] if bias is not None else [])
        gpu.launch(gpu.pipeline(desc), r, m)
        gpu.sync()
        got = b.get(r[1], np.uint32, (m, 2 * k))
    return got[:, :k], got[:, k:].copy().view(np.float32)


def check(gpu, s, bias=None, odd=0, **kw):
    ids, w = run(gpu, s, bias, odd, **kw)
    want, ww = route(hb.bf16_to_f32(s) if s.dtype == np.uint16 else s, bias, **kw)
    assert np.array_equal(ids, want), np.nonzero((ids != want).any(1))[0][:5]
    off = np.abs(w - ww)
    assert (off <= REL * np.abs(ww) + 2.0 ** -140).all(), (off / np.maximum(np.abs(ww), 1e-30)).max()


def scores(seed, m, e, f32, std=1.5):
    s = np.random.default_rng(seed).normal(0, std, (m, e)).astype(np.float32)
    return s if f32 else hb.f32_to_bf16(s)


SCORES = list(hb.Score)


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("e,k", [(1, 1), (2, 2), (7, 3), (64, 6), (65, 1), (100, 10), (128, 8), (256, 8), (384, 32), (512, 10), (1000, 9), (1024, 8)])
def test_experts(gpu, score, f32, e, k):
    check(gpu, scores(e + k, 9, e, f32), odd=1, score=score, top_k=k)


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("group_top", [1, 2])
@pytest.mark.parametrize("e,k,g,t", [(256, 8, 8, 4), (160, 6, 8, 3), (64, 4, 64, 20), (60, 5, 3, 2), (96, 7, 4, 4), (1000, 8, 5, 1), (8, 2, 4, 1), (8, 3, 8, 3)])
def test_groups(gpu, score, with_bias, group_top, e, k, g, t):
    bias = np.random.default_rng(e).normal(0, 0.1, e).astype(np.float32) if with_bias else None
    for f32 in (False, True):
        check(gpu, scores(e + g, 33, e, f32), bias, score=score, top_k=k, groups=g, top_groups=t, group_top=group_top)


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("scale", [1.0, 2.5, -0.5])
def test_weights(gpu, score, renorm, scale):
    for e in (72, 256):
        check(gpu, scores(e, 50, e, True), score=score, top_k=5, renorm=renorm, scale=scale)
        check(gpu, scores(e, 50, e, True), np.linspace(-0.2, 0.2, e).astype(np.float32), score=score, top_k=5, renorm=renorm, scale=scale)


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("with_bias", [False, True])
def test_ties(gpu, score, with_bias):
    """Few distinct scores and biases: the lowest indexes, of groups too."""
    rng = np.random.default_rng(1)
    s = hb.f32_to_bf16(rng.integers(0, 3, (200, 128)).astype(np.float32))
    s[::3] ^= 0x8000  # zeros of both signs
    bias = rng.integers(0, 2, 128).astype(np.float32) if with_bias else None
    check(gpu, s, bias, score=score, top_k=8)
    for group_top in (1, 2):
        check(gpu, s, bias, score=score, top_k=8, groups=16, top_groups=5, group_top=group_top)


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("f32", [False, True])
def test_masked(gpu, score, with_bias, f32):
    """Scores of -inf and NaN, down to rows that leave fewer than top_k experts, or none."""
    rng = np.random.default_rng(2)
    e = 96
    s = rng.normal(0, 1, (e + 4, e)).astype(np.float32)
    for i in range(e):
        s[i, rng.choice(e, i + 1, replace=False)] = -np.inf
    s[e] = np.nan
    s[e + 1, ::2] = np.nan
    s[e + 2, 5], s[e + 2, 50] = np.inf, np.inf
    s[e + 3] = -np.inf
    s[e + 3, 95] = 1.0
    bias = rng.normal(0, 0.1, e).astype(np.float32) if with_bias else None
    s = s if f32 else hb.f32_to_bf16(s)
    for renorm in (False, True):
        check(gpu, s, bias, score=score, top_k=6, renorm=renorm)
        check(gpu, s, bias, score=score, top_k=6, renorm=renorm, groups=8, top_groups=2, group_top=2)
        check(gpu, s, bias, score=score, top_k=6, renorm=renorm, groups=8, top_groups=2, group_top=1)


def test_far_scores(gpu):
    """Large scores of either sign, and biases that are not finite."""
    rng = np.random.default_rng(3)
    s = (rng.normal(0, 1, (64, 64)) * np.exp2(rng.integers(-20, 7, (64, 64)))).astype(np.float32)
    for score in SCORES:
        check(gpu, s, score=score, top_k=4)
    bias = rng.normal(0, 0.1, 64).astype(np.float32)
    bias[3], bias[9], bias[30] = np.inf, -np.inf, np.nan
    check(gpu, scores(1, 20, 64, True), bias, score=hb.Score.Sigmoid, top_k=4)


def test_many_rows_and_repeats(gpu):
    bias = np.random.default_rng(9).normal(0, 0.05, 256).astype(np.float32)
    s = scores(4, 3001, 256, True)
    kw = dict(score=hb.Score.Sigmoid, top_k=8, groups=8, top_groups=4, group_top=2, scale=2.5)
    check(gpu, s, bias, **kw)
    a, b = run(gpu, s, bias, **kw), run(gpu, s, bias, **kw)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1].view(np.uint32), b[1].view(np.uint32))
