"""The 8-bit GEMM with sums in f32 for outputs of two bytes, the SwiGLU and the
routed experts: products far apart in size, whose small ones the f8 MFMA would
cut, exactly; ordinary ones within the bound of f32 additions."""
import numpy as np
import pytest

import f8_ref as f8
import herbert_hip as hb
from test_gpu_f8 import Bufs, marked, run
from test_gpu_f8_forms import F32, SWIGLU, gemm, swiglu_close
from test_gpu_f8_gemm import tables

pytestmark = pytest.mark.gpu


def wide(seed, m, k, n, power=0):
    """x and W whose sums over up to 1152 are whole (times 2^power), and the sums."""
    rng = np.random.default_rng(seed)
    codes, scales = f8.wide_weights(rng, n, k)
    scales = scales * np.float32(2.0 ** power)
    x = f8.exact_x(rng, m, k, (0, 1))
    return codes, scales, x, f8.f64(x) @ f8.values(codes, scales).T


@pytest.mark.parametrize("tile", [{}, dict(ksplit=1), dict(ksplit=3)] + F32)
@pytest.mark.parametrize("out", [hb.Out.Bf16, hb.Out.Residual])
@pytest.mark.parametrize("m,k,n", [(17, 1152, 70), (133, 400, 264)])
def test_exact(gpu, out, m, k, n, tile):
    codes, scales, x, want = wide(m, m, k, n)
    y0 = hb.f32_to_bf16(np.round(8 * np.random.default_rng(m).normal(0, 1, (m, n))).astype(np.float32))
    if out == hb.Out.Residual:
        want = want + f8.f64(y0)
    assert np.abs(want).max() < 2 ** 24
    got = gemm(gpu, codes, scales, x, out, y0, f32_sums=True, rows=m, **tile)
    np.testing.assert_array_equal(got, hb.f32_to_bf16(want.astype(np.float32)))


@pytest.mark.parametrize("tile", [{}] + SWIGLU)
@pytest.mark.parametrize("m,k,n", [(3, 1152, 256), (150, 784, 512)])
def test_exact_swiglu(gpu, m, k, n, tile):
    """Gate and up sums of some 2^-10 of their largest products: h as from the exact ones."""
    codes, scales, x, want = wide(n, m, k, n, -20)
    raw = gemm(gpu, codes, scales, x, hb.Out.Swiglu, marked((m, hb.f8_row_bytes(n // 2))), f32_sums=True, rows=m, **tile)
    swiglu_close(raw, m, n // 2, want)


@pytest.mark.parametrize("out", list(hb.Out))
def test_random(gpu, out):
    m, k, n = 300, 2064, 768
    rng = np.random.default_rng(int(out))
    codes, scales = f8.random_weights(rng, n, k)
    x = hb.normal_bf16(4, 1.0, (m, k))
    xv, wv = f8.row_values(*f8.quantize_rows(x)), f8.values(codes, scales)
    want, bound = xv @ wv.T, f8.sum_bound(xv, wv)
    if out == hb.Out.Swiglu:
        raw = gemm(gpu, codes, scales, x, out, marked((m, hb.f8_row_bytes(n // 2))), f32_sums=True, rows=m)
        return swiglu_close(raw, m, n // 2, want, bound)
    y0 = np.zeros((m, n), np.float32) if out == hb.Out.F32 else hb.normal_bf16(5, 1.0, (m, n))
    if out == hb.Out.Residual:
        want = want + f8.f64(y0)
        bound = bound + f8.U * np.abs(want)
    got = gemm(gpu, codes, scales, x, out, y0, f32_sums=True, rows=m)
    f8.close(got, want, bound, "gemm_f8")
    if out == hb.Out.F32:
        assert np.array_equal(got, gemm(gpu, codes, scales, x, out, y0, rows=m))


@pytest.mark.parametrize("bm", [16, 32, 64, 128])
def test_experts(gpu, bm):
    """Down rows exactly, gate and up's h as from exact sums: the same accuracy at every tile size."""
    hidden, inter, top_k, experts, t = 256, 128, 2, 4, 70
    rng = np.random.default_rng(bm)
    flat, order, tiles = tables(rng, t, top_k, experts, bm, False)
    pairs, mv = t * top_k, bm == 16
    gu = [f8.wide_weights(rng, 2 * inter, hidden) for _ in range(experts)]
    gu = [(c, s * np.float32(2.0 ** -20)) for c, s in gu]
    dn = [f8.wide_weights(rng, hidden, inter) for _ in range(experts)]
    x, hx = f8.exact_x(rng, t, hidden, (0, 1)), f8.exact_x(rng, pairs, inter, (0, 1))

    def rows8(v):
        return v if mv else f8.pack_rows(*f8.quantize_rows(v))

    hrow = 2 * inter if mv else hb.f8_row_bytes(inter)
    with Bufs(gpu) as b:
        st, ls, tl = b.put(np.array([0, 0, 0, t], np.uint32)), b.put(order), b.put(tiles)
        wg, wd = b.put(np.concatenate([f8.pack(*w) for w in gu])), b.put(np.concatenate([f8.pack(*w) for w in dn]))
        h, y = b.put(marked((pairs, hrow))), b.put(marked((pairs, hidden), np.uint16))
        run(gpu, hb.experts_f8(hidden, 2 * inter, hb.Out.Swiglu, hb.Rows.Gather, top_k, experts, t, bm, f32_sums=True),
            [st, wg, b.put(rows8(x)), h, ls, tl], t)
        run(gpu, hb.experts_f8(inter, hidden, hb.Out.Bf16, hb.Rows.Scatter, top_k, experts, t, bm, f32_sums=True),
            [st, wd, b.put(rows8(hx)), y, ls, tl], t)
        hraw, got = b.get(h, np.uint8, (pairs, hrow)), b.get(y, np.uint16, (pairs, hidden))
    for p in range(pairs):
        e = flat[order[p]]
        want = f8.f64(hx[p]) @ f8.values(*dn[e]).T
        np.testing.assert_array_equal(got[order[p]], hb.f32_to_bf16(want.astype(np.float32)))
        s = (f8.f64(x[order[p] // top_k]) @ f8.values(*gu[e]).T)[None]
        if mv:
            g, u = s[:, :inter], s[:, inter:]
            f8.close(np.ascontiguousarray(hraw[p:p + 1]).view(np.uint16), f8.silu(g) * u, f8.swiglu_bound(g, u, 0.0, 0.0), "h")
        else:
            swiglu_close(hraw[p:p + 1], 1, inter, s)
