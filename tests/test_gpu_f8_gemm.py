"""The 8-bit GEMM on the GPU: dense rows and the routed experts, exactly where
every sum is exact in f32 and within a bound from its additions elsewhere, and
its SwiGLU's f8 rows."""
import numpy as np
import pytest

import f8_ref as f8
import herbert_hip as hb
from test_gpu_f8 import Bufs, marked, run

pytestmark = pytest.mark.gpu


def gemm(gpu, codes, scales, x, out, m=None, launch=None, y0=None, **form):
    """Y of the first m rows of x (the launch's rows x's own, or `launch`), rows behind them marked."""
    rows, k = x.shape
    m, n = rows if m is None else m, codes.shape[0]
    if out == hb.Out.Swiglu:
        y = marked((rows, hb.f8_row_bytes(n // 2)))
    else:
        y = np.full((rows, n), 0x4242, np.float32 if out == hb.Out.F32 else np.uint16) if y0 is None else y0
    with Bufs(gpu) as b:
        st, w, yr = b.put(np.array([0, 0, 0, m], np.uint32)), b.put(f8.pack(codes, scales)), b.put(y)
        xr = b.put(f8.pack_rows(*f8.quantize_rows(x)))
        run(gpu, hb.gemm_f8(k, n, out, **form), [st, w, xr, yr, st, st], launch or rows)
        got = b.get(yr, y.dtype, y.shape)
    assert np.array_equal(got[m:], y[m:])
    return got[:m]


def check_h(raw, m, n, want, bound):
    """f8 rows of h within what f32 sums, a rounding to bf16 and one to e4m3 may be off by."""
    codes, scales = f8.unpack_rows(raw, m, n)
    got = f8.row_values(codes, scales)
    near = f8.HALF_BF16 * (np.abs(want) + bound) + bound + 2.0 ** -134
    low, high = f8._groups(np.maximum(np.abs(want) - near, 0), 1), f8._groups(np.abs(want) + near, 1)
    low, high = (np.maximum(t.reshape(m, -1, 128).max(2), f8.TINY) / 448 for t in (low, high))
    assert (scales >= low * (1 - f8.U)).all() and (scales <= high * (1 + f8.U)).all()
    # Half a step: 2^-4 of the value, and 2^-10 of the scale below 2^-6 of it.
    s = np.repeat(scales.astype(np.float64), 128, 1)[:, :n]
    off = np.abs(got - want)
    assert (off <= near + np.maximum(2.0 ** -4 * (np.abs(want) + near), 2.0 ** -10 * s) + f8.U * np.abs(want)).all(), off.max()


def check(gpu, codes, scales, x, out, seed=0, **form):
    n = codes.shape[0]
    xv, wv = f8.row_values(*f8.quantize_rows(x)), f8.values(codes, scales)
    want, bound = xv @ wv.T, (f8.sum_bound if out == hb.Out.F32 else f8.mfma_bound)(xv, wv)
    y0 = hb.normal_bf16(seed + 9, 1.0, want.shape) if out == hb.Out.Residual else None
    got = gemm(gpu, codes, scales, x, out, y0=y0, **form)
    if out == hb.Out.Swiglu:
        g, u, eg, eu = want[:, :n // 2], want[:, n // 2:], bound[:, :n // 2], bound[:, n // 2:]
        return check_h(got, len(x), n // 2, f8.silu(g) * u, f8.swiglu_bound(g, u, eg, eu))
    if out == hb.Out.Residual:
        want = want + f8.f64(y0)
        bound = bound + f8.U * np.abs(want)
    f8.close(got, want, bound, "gemm_f8")


TILES = [dict(bm=32, bn=128), dict(bm=64, bn=128), dict(bm=128, bn=128), dict(bm=128, bn=64, wm=4, wn=1), dict(bm=64, bn=192, wm=1, wn=4),
         dict(bm=256, bn=128, wm=4, wn=2), dict(bm=32, bn=32, wm=1, wn=2, stages=4), dict(bm=128, bn=256, wm=2, wn=4, stages=2)]


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("m,k,n", [(1, 16, 1), (33, 144, 70), (128, 1152, 256), (257, 2192, 333), (70, 3000 // 16 * 16, 515)])
def test_exact(gpu, tile, m, k, n):
    rng = np.random.default_rng(m + k + n)
    codes, scales = f8.exact_weights(rng, n, k)
    x = f8.exact_x(rng, m, k)
    want = f8.f64(x) @ f8.values(codes, scales).T
    assert np.abs(want).max() * 16 < 2 ** 24
    got = gemm(gpu, codes, scales, x, hb.Out.F32, **tile)
    assert np.array_equal(got.astype(np.float64), want)


AHEAD = [dict(bm=256, bn=256, wm=4, wn=2, stages=2, sched=1), dict(bm=128, bn=256, wm=4, wn=2, stages=2, sched=1),
         dict(bm=64, bn=128, wm=2, wn=2, stages=2, sched=1), dict(bm=32, bn=64, wm=1, wn=4, stages=3)]


@pytest.mark.parametrize("tile", TILES + AHEAD + [dict(ksplit=3)])
@pytest.mark.parametrize("out", [hb.Out.Bf16, hb.Out.Residual])
@pytest.mark.parametrize("m,k,n", [(1, 16, 1), (33, 144, 70), (257, 2192, 332)])
def test_exact_bf16(gpu, tile, out, m, k, n):
    """Products within 12 bits of each other, of which the f8 MFMA cuts none: the
    exact sums, rounded once."""
    if "ksplit" in tile and k < 1000:
        pytest.skip("a K tile a part")
    rng = np.random.default_rng(m + k + n)
    codes, scales = f8.exact_weights(rng, n, k)
    x = f8.exact_x(rng, m, k)
    want = f8.f64(x) @ f8.values(codes, scales).T
    y0 = None
    if out == hb.Out.Residual:
        y0 = hb.normal_bf16(m, 8.0, want.shape)
        y0 = hb.f32_to_bf16(np.round(hb.bf16_to_f32(y0)).astype(np.float32))  # wholes: the sum is exact too
        want = want + f8.f64(y0)
    assert np.array_equal(gemm(gpu, codes, scales, x, out, y0=y0, **tile), hb.f32_to_bf16(want.astype(np.float32)))


SWIGLU = [dict(bm=256, wm=4, wn=2, stages=2), dict(bm=128, wm=2, wn=4, stages=3), dict(bm=64, wm=1, wn=8, stages=3), dict(bm=32, wm=1, wn=8, stages=4),
          dict(bm=32, wm=2, wn=4, stages=2, sched=1)]


@pytest.mark.parametrize("tile", SWIGLU)
@pytest.mark.parametrize("m,k,n", [(1, 16, 256), (300, 400, 768)])
def test_exact_swiglu(gpu, tile, m, k, n):
    """Exact sums under the SwiGLU: h within its own roundings."""
    rng = np.random.default_rng(m + k + n)
    codes, scales = f8.exact_weights(rng, n, k)
    scales = scales * np.float32(2.0 ** -10)  # sums around 1
    x = f8.exact_x(rng, m, k)
    s = f8.f64(x) @ f8.values(codes, scales).T
    g, u = s[:, :n // 2], s[:, n // 2:]
    got = gemm(gpu, codes, scales, x, hb.Out.Swiglu, bn=256, **tile)
    check_h(got, m, n // 2, f8.silu(g) * u, f8.swiglu_bound(g, u, 0.0, 0.0))


@pytest.mark.parametrize("m,k,n,ksplit", [(17, 1152, 70, 0), (50, 400, 300, 2), (300, 1152, 515, 0)])
def test_wide_products(gpu, m, k, n, ksplit):
    """Products far apart in size: the small ones stay in an f32 output's sums."""
    rng = np.random.default_rng(m + n)
    codes, scales = f8.wide_weights(rng, n, k)
    x = f8.exact_x(rng, m, k, (0, 1))
    want = f8.f64(x) @ f8.values(codes, scales).T
    assert np.array_equal(gemm(gpu, codes, scales, x, hb.Out.F32, rows=m, **(dict(ksplit=ksplit) if ksplit else {})).astype(np.float64), want)


@pytest.mark.parametrize("out", list(hb.Out))
@pytest.mark.parametrize("m,k,n", [(17, 2560, 512), (200, 1040, 768), (513, 2064, 1280)])
def test_outs(gpu, out, m, k, n):
    rng = np.random.default_rng(m + n)
    codes, scales = f8.random_weights(rng, n, k)
    check(gpu, codes, scales, hb.normal_bf16(m, 1.0, (m, k)), out, rows=m)


@pytest.mark.parametrize("out", [hb.Out.Bf16, hb.Out.F32, hb.Out.Residual])
@pytest.mark.parametrize("n", [333, 1002, 1003])
def test_ragged_columns(gpu, out, n):
    rng = np.random.default_rng(n)
    codes, scales = f8.random_weights(rng, n, 784)
    check(gpu, codes, scales, hb.normal_bf16(n, 1.0, (150, 784)), out, rows=150)


@pytest.mark.parametrize("parts", [2, 3, 8])
@pytest.mark.parametrize("out", [hb.Out.Bf16, hb.Out.F32, hb.Out.Residual])
def test_split_k(gpu, parts, out):
    rng = np.random.default_rng(parts)
    codes, scales = f8.random_weights(rng, 300, 2704)
    check(gpu, codes, scales, hb.normal_bf16(parts, 1.0, (50, 2704)), out, rows=50, ksplit=parts)


@pytest.mark.parametrize("n", [1, 3, 301, 334])
@pytest.mark.parametrize("out", [hb.Out.Bf16, hb.Out.F32, hb.Out.Residual])
def test_split_k_ragged(gpu, out, n):
    """Any N and fewer rows than launched: exact sums, the rows behind left as they are."""
    rng = np.random.default_rng(n)
    codes, scales = f8.exact_weights(rng, n, 1040)
    x = f8.exact_x(rng, 53, 1040)
    want = f8.f64(x) @ f8.values(codes, scales).T
    for m in (53, 31):
        y0 = np.zeros(want.shape, np.uint16) if out == hb.Out.Residual else None
        got = gemm(gpu, codes, scales, x, out, m=m, y0=y0, rows=53, ksplit=4)
        exact = want[:m].astype(np.float32)
        assert np.array_equal(got, exact if out == hb.Out.F32 else hb.f32_to_bf16(exact + np.float32(0)))


@pytest.mark.parametrize("out", [hb.Out.Bf16, hb.Out.Swiglu])
def test_fewer_rows_than_launched(gpu, out):
    """state[3] below the launch's rows: the rows behind stay as they are."""
    rng = np.random.default_rng(1)
    codes, scales = f8.random_weights(rng, 512, 640)
    x = hb.normal_bf16(1, 1.0, (300, 640))
    whole = gemm(gpu, codes, scales, x, out, rows=300)
    for m in (1, 127, 128, 129, 299):
        assert np.array_equal(gemm(gpu, codes, scales, x, out, m=m, rows=300), whole[:m])
    assert gemm(gpu, codes, scales, x, out, m=0, rows=300).size == 0


def test_rows_apart(gpu):
    """A row with a NaN or an infinity leaves the others alone; so does a NaN weight."""
    rng = np.random.default_rng(3)
    k, n = 1040, 272
    codes, scales = f8.random_weights(rng, n, k)
    x = hb.normal_bf16(4, 1.0, (140, k))
    whole = gemm(gpu, codes, scales, x, hb.Out.F32)
    x[5, 77], x[131, 1039], x[12] = 0x7FC0, 0x7F80, 0
    got = gemm(gpu, codes, scales, x, hb.Out.F32)
    assert np.isnan(got[5]).all() and np.isnan(got[131]).all() and (got[12] == 0).all()
    rest = [i for i in range(140) if i not in (5, 131, 12)]
    assert np.array_equal(got[rest], whole[rest])
    codes[100, 3] = 0x7F
    got = gemm(gpu, codes, scales, x, hb.Out.F32)
    assert np.isnan(got[:, 100]).all() and np.array_equal(got[rest][:, np.arange(n) != 100], whole[rest][:, np.arange(n) != 100])


def test_swiglu_nan_and_zero_rows(gpu):
    rng = np.random.default_rng(5)
    codes, scales = f8.random_weights(rng, 512, 256)
    x = hb.normal_bf16(6, 1.0, (40, 256))
    x[3], x[7, 9] = 0, 0x7FC0
    raw = gemm(gpu, codes, scales, x, hb.Out.Swiglu)
    c, s = f8.unpack_rows(raw, 40, 256)
    assert (f8.row_values(c, s)[3] == 0).all() and np.isnan(f8.row_values(c, s)[7]).all()
    rest = [i for i in range(40) if i not in (3, 7)]
    assert np.isfinite(f8.row_values(c, s)[rest]).all()


# ---- the routed experts ----

def tables(rng, t, top_k, experts, bm, skew):
    """A random route's sorted pairs and the tile table that moe_sort makes of them."""
    p = np.exp(-np.arange(experts) / 4.0) if skew else np.ones(experts)
    ids = np.array([np.sort(rng.choice(experts, top_k, replace=False, p=p / p.sum())) for _ in range(t)])
    flat = ids.reshape(-1)
    order = np.argsort(flat, kind="stable")
    tab, at = [], 0
    for e in range(experts):
        c = int((flat == e).sum())
        for j in range(0, c, bm):
            tab.append((e, at + j, min(bm, c - j)))
        at += c
    room = hb.moe_tiles(t, top_k, experts, bm)
    tiles = np.full(1 + 3 * room, 0xFFFFFFFF, np.uint32)
    tiles[0] = len(tab)
    tiles[1:1 + 3 * len(tab)] = np.array(tab, np.uint32).reshape(-1)
    return flat, order.astype(np.uint32), tiles


@pytest.mark.parametrize("t,bm,skew", [(1, 16, False), (9, 16, True), (40, 16, False), (40, 32, False), (60, 64, True), (100, 128, True)])
def test_experts(gpu, t, bm, skew):
    """Gate and up with the SwiGLU over gathered rows, down over scattered ones,
    in the forms of both tile sizes: h of each pair, and y of the h there is."""
    hidden, inter, top_k, experts = 400, 256, 3, 10
    rng = np.random.default_rng(t + bm)
    flat, order, tiles = tables(rng, t, top_k, experts, bm, skew)
    pairs, mv = t * top_k, bm == 16
    gu = [f8.random_weights(rng, 2 * inter, hidden) for _ in range(experts)]
    dn = [f8.random_weights(rng, hidden, inter) for _ in range(experts)]
    x = hb.normal_bf16(t, 1.0, (t, hidden))
    hrow = 2 * inter if mv else hb.f8_row_bytes(inter)
    with Bufs(gpu) as b:
        st, ls, tl = b.put(np.array([0, 0, 0, t], np.uint32)), b.put(order), b.put(tiles)
        wg, wd = b.put(np.concatenate([f8.pack(*w) for w in gu])), b.put(np.concatenate([f8.pack(*w) for w in dn]))
        xr = b.put(x) if mv else b.put(f8.pack_rows(*f8.quantize_rows(x)))
        h, y = b.put(marked((pairs, hrow))), b.put(marked((pairs, hidden), np.uint16))
        run(gpu, hb.experts_f8(hidden, 2 * inter, hb.Out.Swiglu, hb.Rows.Gather, top_k, experts, t, bm), [st, wg, xr, h, ls, tl], t)
        run(gpu, hb.experts_f8(inter, hidden, hb.Out.Bf16, hb.Rows.Scatter, top_k, experts, t, bm), [st, wd, h, y, ls, tl], t)
        hraw, got = b.get(h, np.uint8, (pairs, hrow)), b.get(y, np.uint16, (pairs, hidden))
    xv = f8.row_values(*f8.quantize_rows(x))
    for p in range(pairs):
        e, r = flat[order[p]], order[p] // top_k
        wv, row = f8.values(*gu[e]), xv[r:r + 1]
        bound_of = f8.sum_bound if mv else f8.mfma_bound
        s, eb = row @ wv.T, bound_of(row, wv)
        g, u = s[:, :inter], s[:, inter:]
        want, bound = f8.silu(g) * u, f8.swiglu_bound(g, u, eb[:, :inter], eb[:, inter:])
        if mv:
            hbits = hraw[p:p + 1].view(np.uint16)
            f8.close(hbits, want, bound, "h")
            hv = f8.row_values(*f8.quantize_rows(hbits))
        else:
            check_h(hraw[p:p + 1], 1, inter, want, bound)
            hv = f8.row_values(*f8.unpack_rows(hraw[p:p + 1], 1, inter))
        dv = f8.values(*dn[e])
        f8.close(got[order[p]:order[p] + 1], hv @ dv.T, bound_of(hv, dv), "y")


@pytest.mark.parametrize("bm", [16, 64])
def test_experts_fewer_rows(gpu, bm):
    """Tiles past the rows of state[3] and experts past the last write nothing."""
    hidden, inter, top_k, experts, t = 256, 128, 2, 8, 12
    rng = np.random.default_rng(bm)
    flat, order, tiles = tables(rng, t, top_k, experts, bm, False)
    w = np.concatenate([f8.pack(*f8.random_weights(rng, hidden, inter)) for _ in range(experts)])
    x = hb.normal_bf16(1, 1.0, (t * top_k, inter))
    m = 5
    with Bufs(gpu) as b:
        st, ls, tl, wr = b.put(np.array([0, 0, 0, m], np.uint32)), b.put(order), b.put(tiles), b.put(w)
        xr, y = b.put(x if bm == 16 else f8.pack_rows(*f8.quantize_rows(x))), b.put(marked((t * top_k, hidden), np.uint16))
        run(gpu, hb.experts_f8(inter, hidden, hb.Out.Bf16, hb.Rows.Scatter, top_k, experts, t, bm), [st, wr, xr, y, ls, tl], t)
        got = b.get(y, np.uint16, (t * top_k, hidden))
    # Sorted rows from m * top_k on are none of the block's; list entries past
    # them come to its last row.
    assert (got[m * top_k:] == 0x5A5A).all()
