"""block_norm on the GPU against its formulas in 64 bits: the post norm, each
gate, the scales and the pre norm, rows of any length, odd offsets, outputs
over their inputs."""
import numpy as np
import pytest

import herbert_hip as hb

pytestmark = pytest.mark.gpu

EPS = 1e-6
# f32 arithmetic: a row's sum of squares takes at most 8 * 4 additions a
# thread, 6 in the wave and 15 over waves, half of which reaches the root;
# then some ten roundings of half a step each.
REL = (53 / 2 + 12) * 2.0 ** -24
HALF = 2.0 ** -8  # one rounding to bf16


def f64(bits):
    return hb.bf16_to_f32(bits).astype(np.float64)


def rms(t, w, plus_one):
    return t / np.sqrt((t * t).mean(-1, keepdims=True) + EPS) * (f64(w) + (1 if plus_one else 0))


def reference(x, y, plus_one, post=None, gate=hb.Gate.Off, g=None, scales=None):
    """(xo, what its f32 terms sum to in size)."""
    a, v = f64(x), f64(y)
    if post is not None:
        v = rms(v, post, plus_one)
    if gate in (hb.Gate.Rows, hb.Gate.Elements):
        s = 1 / (1 + np.exp(-f64(g)))
        v = v * (s[:, None] if gate == hb.Gate.Rows else s)
    if gate == hb.Gate.Channels:
        v = v * f64(g)
    if scales is not None:
        a, v = a * np.float64(scales[0]), v * np.float64(scales[1])
    return a + v, np.abs(a) + np.abs(v)


def check(gpu, n, m, post, pre, gate, scales, plus_one, odd=0, over=None, seed=0):
    rng = np.random.default_rng(n * 31 + m + seed)
    x, y = hb.normal_bf16(n + seed, 2.0, (m, n)), hb.normal_bf16(n + 1 + seed, 0.5, (m, n))
    w_post, w_pre = hb.normal_bf16(3, 0.5, n), hb.normal_bf16(4, 0.5, n)
    shape = {hb.Gate.Off: None, hb.Gate.Rows: m, hb.Gate.Elements: (m, n), hb.Gate.Channels: n}[gate]
    g = hb.normal_bf16(5, 2.0, shape) if shape else None
    sc = rng.uniform(0.5, 1.5, 2).astype(np.float32) if scales else None
    bufs = {}

    def put(name, a):
        pad = odd if a.dtype == np.uint16 else 0
        mark = np.full(pad + a.size + 7, 0x4242, a.dtype)
        mark[pad:pad + a.size] = a.reshape(-1)
        bufs[name] = gpu.alloc_with(mark)
        return hb.r(bufs[name], pad * a.dtype.itemsize)

    def get(rng_, name):
        a = gpu.download(bufs[name], np.uint16, odd + m * n + 7)
        assert (a[:odd] == 0x4242).all() and (a[-7:] == 0x4242).all(), name
        return a[odd:odd + m * n].reshape(m, n)

    try:
        r = {"x": put("x", x), "y": put("y", y)}
        if gate == hb.Gate.Elements:
            r["gate"] = put("gate", g)
        names = {"xo": "xo", "h": "h", **(over or {})}
        for o in ("xo", "h"):
            if names[o] == o:
                r[o] = put(o, np.full((m, n), 0x1111, np.uint16))
            else:
                r[o] = r[names[o]]
        ranges = [r["x"], r["y"], r["xo"]] + ([r["h"]] if pre else []) + ([put("w_post", w_post)] if post else [])
        if gate != hb.Gate.Off:
            ranges.append(r["gate"] if gate == hb.Gate.Elements else put("gate", g))
        ranges += ([put("scales", sc)] if scales else []) + ([put("w_pre", w_pre)] if pre else [])
        gpu.launch(gpu.pipeline(hb.block_norm(n, EPS, plus_one, post, pre, gate, scales)), ranges, m)
        gpu.sync()
        xo = get(r, names["xo"])
        want, size = reference(x, y, plus_one, w_post if post else None, gate, g, sc)
        off = np.abs(f64(xo) - want)
        assert (off <= HALF * np.abs(want) + (1 + HALF) * 2 * REL * size + 2.0 ** -134).all(), off.max()
        if pre:
            h = get(r, names["h"])
            want = rms(f64(xo), w_pre, plus_one)
            off = np.abs(f64(h) - want)
            assert (off <= (HALF + 2 * REL) * np.abs(want) + 2.0 ** -134).all(), off.max()
    finally:
        for b in bufs.values():
            gpu.free(b)


GATES = list(hb.Gate)


@pytest.mark.parametrize("n", [1, 7, 8, 9, 64, 511, 513, 2560, 2565, 8192, 8200, 20001, 32768])
@pytest.mark.parametrize("gate", GATES)
def test_lengths(gpu, n, gate):
    check(gpu, n, 3, True, True, gate, True, True, odd=n % 2)


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("pre", [False, True])
@pytest.mark.parametrize("scales", [False, True])
@pytest.mark.parametrize("gate", GATES)
def test_parts(gpu, post, pre, scales, gate):
    check(gpu, 520, 5, post, pre, gate, scales, False, odd=1)


@pytest.mark.parametrize("over", [{"xo": "x"}, {"xo": "y"}, {"xo": "x", "h": "y"}, {"xo": "y", "h": "x"},
                                  {"xo": "x", "h": "gate"}])
def test_outputs_over_inputs(gpu, over):
    check(gpu, 2563, 4, True, True, hb.Gate.Elements, False, True, over=over)


def test_many_rows(gpu):
    check(gpu, 5120, 1025, True, True, hb.Gate.Rows, True, True)


def test_zero_rows_and_non_finite(gpu):
    """A row of zeros norms to zeros; a NaN stays in its row."""
    n = 264
    x = np.zeros((3, n), np.uint16)
    x[2] = hb.normal_bf16(1, 1.0, n)
    y = np.zeros((3, n), np.uint16)
    y[1, 5] = 0x7FC0
    w = hb.normal_bf16(2, 1.0, n)
    bufs = [gpu.alloc_with(a) for a in (x, y, x, x, w, w)]
    try:
        gpu.launch(gpu.pipeline(hb.block_norm(n, EPS, False, True, True)), [hb.r(b) for b in bufs], 3)
        gpu.sync()
        xo, h = (f64(gpu.download(b, np.uint16, 3 * n).reshape(3, n)) for b in bufs[2:4])
    finally:
        for b in bufs:
            gpu.free(b)
    assert (xo[0] == 0).all() and (h[0] == 0).all()
    assert np.isnan(xo[1]).all() and np.isnan(h[1]).all()
    assert np.array_equal(xo[2], f64(x[2])) and np.isfinite(h[2]).all()
