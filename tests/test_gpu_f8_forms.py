"""The forms of the 8-bit GEMM that its defaults take, each over shapes that none
of them divides, and outputs at any element of a buffer: exactly where every sum
is exact in f32, and within a bound from its additions elsewhere."""
import numpy as np
import pytest

import f8_ref as f8
import herbert_hip as hb
from test_gpu_f8 import Bufs, run

pytestmark = pytest.mark.gpu


def form(bm, bn, wm, wn, stages, sched):
    return dict(bm=bm, bn=bn, wm=wm, wn=wn, stages=stages, sched=sched)


def gemm(gpu, codes, scales, x, out, y0, odd=0, **form):
    """Y over y0, at `odd` elements of its buffer, nothing written around it."""
    (m, k), n = x.shape, codes.shape[0]
    with Bufs(gpu) as b:
        st, w = b.put(np.array([0, 0, 0, m], np.uint32)), b.put(f8.pack(codes, scales))
        xr, y = b.put(f8.pack_rows(*f8.quantize_rows(x))), b.put(y0, odd)
        run(gpu, hb.gemm_f8(k, n, out, **form), [st, w, xr, y, st, st], m)
        return b.get(y, y0.dtype, y0.shape)


def exact(gpu, out, m, k, n, odd=0, **form):
    """Sums that f32 holds, and of which the f8 MFMA cuts nothing."""
    rng = np.random.default_rng(m + k + n)
    codes, scales = f8.exact_weights(rng, n, k)
    x = f8.exact_x(rng, m, k)
    want = f8.f64(x) @ f8.values(codes, scales).T
    assert np.abs(want).max() * 16 < 2 ** 24
    if out == hb.Out.F32:
        got = gemm(gpu, codes, scales, x, out, np.full((m, n), 66.0, np.float32), odd, **form)
        return np.testing.assert_array_equal(got, want)
    y0 = hb.normal_bf16(m, 8.0, (m, n))
    if out == hb.Out.Residual:
        y0 = hb.f32_to_bf16(np.round(hb.bf16_to_f32(y0)).astype(np.float32))  # wholes: the sum is exact too
        want = want + f8.f64(y0)
    got = gemm(gpu, codes, scales, x, out, y0, odd, **form)
    np.testing.assert_array_equal(got, hb.f32_to_bf16(want.astype(np.float32)))


@pytest.mark.parametrize("odd", [1, 3, 4, 7])
@pytest.mark.parametrize("tile", [form(32, 32, 1, 2, 4, 0), form(128, 128, 4, 2, 2, 1), dict(bm=64, bn=64, ksplit=2)])
@pytest.mark.parametrize("out,n", [(hb.Out.Bf16, 136), (hb.Out.Bf16, 137), (hb.Out.Bf16, 138), (hb.Out.Residual, 136), (hb.Out.Residual, 138),
                                   (hb.Out.F32, 136), (hb.Out.F32, 137)])
def test_output_at_any_element(gpu, out, n, tile, odd):
    exact(gpu, out, 133, 400, n, odd, **tile)


@pytest.mark.parametrize("odd", [1, 5])
@pytest.mark.parametrize("bm", [16, 32, 64, 128])
def test_experts_output_at_any_element(gpu, bm, odd):
    """Down's scattered rows, whole chunks of eight elements wide."""
    inter, hidden, top_k, experts, t = 128, 264, 2, 3, 50
    rng = np.random.default_rng(bm)
    w = [f8.exact_weights(rng, hidden, inter) for _ in range(experts)]
    pairs = t * top_k
    x, expert = f8.exact_x(rng, pairs, inter), np.sort(rng.integers(0, experts, pairs))
    order = rng.permutation(pairs).astype(np.uint32)
    tab = []
    for e in range(experts):
        first, last = np.searchsorted(expert, [e, e + 1])
        tab += [(e, i, min(bm, last - i)) for i in range(first, last, bm)]
    tiles = np.zeros(1 + 3 * hb.moe_tiles(t, top_k, experts, bm), np.uint32)
    tiles[0] = len(tab)
    tiles[1:1 + 3 * len(tab)] = np.array(tab, np.uint32).reshape(-1)
    with Bufs(gpu) as b:
        st, ls, tl, wr = b.put(np.array([0, 0, 0, t], np.uint32)), b.put(order), b.put(tiles), b.put(np.concatenate([f8.pack(*v) for v in w]))
        xr = b.put(x if bm == 16 else f8.pack_rows(*f8.quantize_rows(x)))
        y = b.put(np.full((pairs, hidden), 0x4242, np.uint16), odd)
        run(gpu, hb.experts_f8(inter, hidden, hb.Out.Bf16, hb.Rows.Scatter, top_k, experts, t, bm), [st, wr, xr, y, ls, tl], t)
        got = b.get(y, np.uint16, (pairs, hidden))
    want = np.zeros((pairs, hidden))
    for p in range(pairs):
        want[order[p]] = f8.f64(x[p]) @ f8.values(*w[expert[p]]).T
    np.testing.assert_array_equal(got, hb.f32_to_bf16(want.astype(np.float32)))
