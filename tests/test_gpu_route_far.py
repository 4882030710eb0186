"""route_topk's sigmoid weights at scores far below 0, against their definition
in 64 bits taken relative to the row's largest chosen score."""
import numpy as np
import pytest

import herbert_hip as hb
from test_gpu_route_topk import REL, run

pytestmark = pytest.mark.gpu


def weights(s, ids, renorm, scale):
    """sigmoid(s) of the chosen, [m][k] in 64 bits: log(sigmoid) = s - log(1 + e^s)."""
    x = np.take_along_axis(s.astype(np.float64), ids.astype(np.int64), 1)
    log = np.where(x > 0, -np.log1p(np.exp(-np.abs(x))), x - np.log1p(np.exp(np.minimum(x, 0))))
    if not renorm:
        return np.exp(log) * scale
    w = np.exp(log - log.max(1, keepdims=True))
    return w / w.sum(1, keepdims=True) * scale


def check(gpu, s, want_ids, bias=None, renorm=True, scale=2.5, **kw):
    ids, w = run(gpu, s, bias, score=hb.Score.Sigmoid, renorm=renorm, scale=scale, **kw)
    assert np.array_equal(ids, want_ids)
    want = weights(hb.bf16_to_f32(s) if s.dtype == np.uint16 else s, ids, renorm, scale)
    off = np.abs(w - want)
    assert (off <= REL * np.abs(want) + 2.0 ** -140).all(), (off / np.maximum(np.abs(want), 1e-30)).max()
    if renorm:
        assert (np.abs(w.sum(1) - scale) <= REL * scale).all()


def largest(c, k):
    return np.sort(np.argsort(-c, axis=1, kind="stable")[:, :k], axis=1)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("top", [-1e-3, -1.0, -20.0, -86.9, -87.1, -88.8, -90.0, -103.5, -200.0, -1000.0, -3e4])
def test_largest(gpu, top, renorm, f32):
    """Rows whose largest score is `top`, the others within 5, 60 and 400 of it."""
    rng = np.random.default_rng(int(-top * 1000) % 2**31)
    s = (top - np.abs(rng.normal(0, 1, (90, 72))) * np.repeat([5.0, 60.0, 400.0], 30)[:, None]).astype(np.float32)
    s[np.arange(90), rng.integers(0, 72, 90)] = top
    bits = s if f32 else hb.f32_to_bf16(s)
    x = s if f32 else hb.bf16_to_f32(bits)
    check(gpu, bits, largest(x, 6), renorm=renorm, top_k=6)


def test_one_expert(gpu):
    """A row's only choice has the whole weight at any finite score."""
    s = np.linspace(-2000, 100, 3000).astype(np.float32)[:, None]
    check(gpu, s, np.zeros((3000, 1), np.uint32), top_k=1)
    check(gpu, np.full((2, 1), -3.4e38, np.float32), np.zeros((2, 1), np.uint32), top_k=1)


@pytest.mark.parametrize("groups", [1, 8])
def test_chosen_by_bias(gpu, groups):
    """Biases that choose experts whose scores all lie below -90, beside rows that
    also have some above 0."""
    rng = np.random.default_rng(groups)
    s = (-90 - np.abs(rng.normal(0, 20, (64, 64)))).astype(np.float32)
    s[::2, :4] = rng.normal(0, 1, (32, 4))
    bias = (8 + rng.permutation(64)).astype(np.float32)  # whole numbers, far apart beside any sigmoid
    c = 1 / (1 + np.exp(-s.astype(np.float64))) + bias
    if groups > 1:
        g = np.sort(c.reshape(64, 8, 8), axis=2)[:, :, -2:].sum(2)
        keep = np.argsort(-g, axis=1, kind="stable")[:, :3]
        stays = (keep[:, :, None] == np.arange(8)).any(1)
        c = np.where(np.repeat(stays, 8, 1), c, -np.inf)
    check(gpu, s, largest(c, 5), bias, top_k=5, groups=groups, top_groups=3 if groups > 1 else 1, group_top=2)
