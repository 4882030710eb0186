"""The forms of the 8-bit matvec that its defaults take, at one to four loads of x
rows, over shapes that no block divides: exactly where every sum is exact in
f32, and the SwiGLU's h as from the exact sums; and the experts' tiles of 256
rows and of a decode batch."""
import numpy as np
import pytest

import f8_ref as f8
import herbert_hip as hb
from test_gpu_f8 import Bufs, marked, matvec, run
from test_gpu_f8_forms import swiglu_close
from test_gpu_f8_gemm import tables

pytestmark = pytest.mark.gpu

# (W rows a wave, waves on K, waves, stages): what the defaults take (tests/test_f8_host_forms.py
# holds them to these); the second holds no more than 8 x rows.
FORMS = [(16, 16, 16, 1), (16, 16, 16, 2), (16, 8, 8, 1), (16, 4, 4, 1), (16, 2, 4, 1), (16, 1, 4, 1), (32, 8, 8, 2), (32, 4, 4, 2), (32, 2, 4, 2),
         (32, 1, 4, 2), (64, 8, 8, 1), (64, 2, 4, 1), (64, 1, 4, 1)]
CASES = [(f, m) for f in FORMS for m in (1, 4, 7, 10, 16) if f != FORMS[1] or m <= 8]


@pytest.mark.parametrize("form,m", CASES)
@pytest.mark.parametrize("out", [hb.Out.F32, hb.Out.Bf16, hb.Out.Residual])
@pytest.mark.parametrize("k,n", [(2064, 333), (272, 1100), (16, 40)])
def test_exact(gpu, form, m, out, k, n):
    rng = np.random.default_rng(m * 1000 + k + n)
    codes, scales = f8.exact_weights(rng, n, k)
    x = f8.exact_x(rng, m, k)
    want = f8.f64(x) @ f8.values(codes, scales).T
    y0 = None
    if out == hb.Out.Residual:
        y0 = hb.f32_to_bf16(np.round(8 * rng.normal(0, 1, want.shape)).astype(np.float32))
        want = want + f8.f64(y0)
    rows, split, waves, unroll = form
    got = matvec(gpu, codes, scales, x, out, y0, m % 2, mv_m=m, rows=rows, split=split, waves=waves, unroll=unroll)
    want = want.astype(np.float32)
    np.testing.assert_array_equal(got, want if out == hb.Out.F32 else hb.f32_to_bf16(want))


@pytest.mark.parametrize("form,m", [c for c in CASES if c[0][0] > 16])
@pytest.mark.parametrize("k,n", [(2064, 512), (16, 1280)])
def test_exact_swiglu(gpu, form, m, k, n):
    rng = np.random.default_rng(m * 1000 + k + n)
    codes, scales = f8.exact_weights(rng, n, k)
    scales = scales * np.float32(2.0 ** -10)  # sums around 1
    x = f8.exact_x(rng, m, k)
    s = f8.f64(x) @ f8.values(codes, scales).T
    rows, split, waves, unroll = form
    got = matvec(gpu, codes, scales, x, hb.Out.Swiglu, mv_m=m, rows=rows, split=split, waves=waves, unroll=unroll)
    g, u = s[:, :n // 2], s[:, n // 2:]
    f8.close(got, f8.silu(g) * u, f8.swiglu_bound(g, u, 0.0, 0.0), "h")


@pytest.mark.parametrize("t,bm,k,n", [(300, 256, 400, 512), (40, 16, 1040, 512), (2, 16, 1040, 512), (2, 16, 272, 256), (2, 16, 144, 256), (2, 16, 128, 256), (60, 16, 272, 512)])
def test_experts(gpu, t, bm, k, n):
    """Gate and up with the SwiGLU over gathered rows, then down's exact sums over scattered ones."""
    top_k, experts = 2, 3
    rng = np.random.default_rng(t + bm + k)
    flat, order, tiles = tables(rng, t, top_k, experts, bm, True)
    pairs, mv = t * top_k, bm == 16
    gu = [f8.exact_weights(rng, n, k) for _ in range(experts)]
    gu = [(c, s * np.float32(2.0 ** -10)) for c, s in gu]
    dn = [f8.exact_weights(rng, n, k) for _ in range(experts)]
    x, hx = f8.exact_x(rng, t, k), f8.exact_x(rng, pairs, k)

    def rows8(v):
        return v if mv else f8.pack_rows(*f8.quantize_rows(v))

    hrow = n if mv else hb.f8_row_bytes(n // 2)
    with Bufs(gpu) as b:
        st, ls, tl = b.put(np.array([0, 0, 0, t], np.uint32)), b.put(order), b.put(tiles)
        wg, wd = b.put(np.concatenate([f8.pack(*w) for w in gu])), b.put(np.concatenate([f8.pack(*w) for w in dn]))
        h, y = b.put(marked((pairs, hrow))), b.put(marked((pairs, n), np.uint16))
        run(gpu, hb.experts_f8(k, n, hb.Out.Swiglu, hb.Rows.Gather, top_k, experts, t, bm), [st, wg, b.put(rows8(x)), h, ls, tl], t)
        run(gpu, hb.experts_f8(k, n, hb.Out.Bf16, hb.Rows.Scatter, top_k, experts, t, bm), [st, wd, b.put(rows8(hx)), y, ls, tl], t)
        hraw, got = b.get(h, np.uint8, (pairs, hrow)), b.get(y, np.uint16, (pairs, n))
    for p in range(pairs):
        e = flat[order[p]]
        want = f8.f64(hx[p]) @ f8.values(*dn[e]).T
        np.testing.assert_array_equal(got[order[p]], hb.f32_to_bf16(want.astype(np.float32)))
        s = (f8.f64(x[order[p] // top_k]) @ f8.values(*gu[e]).T)[None]
        if mv:
            g, u = s[:, :n // 2], s[:, n // 2:]
            f8.close(np.ascontiguousarray(hraw[p:p + 1]).view(np.uint16), f8.silu(g) * u, f8.swiglu_bound(g, u, 0.0, 0.0), "h")
        else:
            swiglu_close(hraw[p:p + 1], 1, n // 2, s)


def test_sorted_tiles_of_256(gpu):
    """moe_sort's table of 256-row tiles is the one that the products read."""
    t, top_k, experts, k, n = 500, 2, 64, 128, 272
    rng = np.random.default_rng(1)
    flat, order, _ = tables(rng, t, top_k, experts, 256, True)
    w = [f8.exact_weights(rng, n, k) for _ in range(experts)]
    x = f8.exact_x(rng, t * top_k, k)
    route = np.zeros((t, 2 * top_k), np.uint32)
    route[:, :top_k] = flat.reshape(t, top_k)
    with Bufs(gpu) as b:
        st, wr, rt = b.put(np.array([0, 0, 0, t], np.uint32)), b.put(np.concatenate([f8.pack(*v) for v in w])), b.put(route)
        ls, tl = b.put(np.zeros(t * top_k, np.uint32)), b.put(np.zeros(1 + 3 * hb.moe_tiles(t, top_k, experts, 256), np.uint32))
        y = b.put(marked((t * top_k, n), np.uint16))
        run(gpu, hb.Desc(kind=hb.Kind.SORT, experts=experts, top_k=top_k, bm=256, rows_max=t), [st, rt, ls, tl], t)
        run(gpu, hb.experts_f8(k, n, hb.Out.Bf16, hb.Rows.Scatter, top_k, experts, t, 256),
            [st, wr, b.put(f8.pack_rows(*f8.quantize_rows(x))), y, ls, tl], t)
        got, sorted_pairs = b.get(y, np.uint16, (t * top_k, n)), b.get(ls, np.uint32, (t * top_k,))
    assert np.array_equal(sorted_pairs, order)
    for p in range(t * top_k):
        want = f8.f64(x[p]) @ f8.values(*w[flat[order[p]]]).T
        np.testing.assert_array_equal(got[order[p]], hb.f32_to_bf16(want.astype(np.float32)))
