"""Weights of 4 bits on the GPU against their definition in 64 bits: quantise,
pack and read back bit for bit, the matvec exactly where every sum is exact
and within the sums' bound elsewhere, the experts over moe_sort's tiles."""
import numpy as np
import pytest

import herbert_hip as hb
import q4_ref as q4

pytestmark = pytest.mark.gpu

GROUPS = [32, 64, 128]
SHAPES = [(8, 1), (32, 16), (136, 17), (128, 48), (1000, 33), (1024, 112), (2568, 50)]


def run(gpu, desc, ranges, m):
    gpu.launch(gpu.pipeline(desc), ranges, m)
    gpu.sync()


@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("k,n", SHAPES)
def test_pack_and_dequantize(gpu, k, n, group):
    """Two matrices packed, read back at an odd offset: bit for bit, and
    nothing written past them."""
    rng = np.random.default_rng(k * n + group)
    codes, scales = q4.random_codes(rng, 2 * n, k, group)
    w = q4.pack(gpu, codes, scales, k, n, group, 2)
    mark = np.full(2 * n * k + 9, 0x4242, np.uint16)
    out = gpu.alloc_with(mark)
    try:
        run(gpu, hb.q4_dequantize(k, n, group), [hb.r(w), hb.r(out, 6)], 2)
        got = gpu.download(out, np.uint16, mark.size)
    finally:
        gpu.free(w)
        gpu.free(out)
    assert np.array_equal(got[3:-6].reshape(2 * n, k), hb.f32_to_bf16(q4.values(codes, scales, group).astype(np.float32)))
    assert (got[:3] == 0x4242).all() and (got[-6:] == 0x4242).all()


def special_rows(w, rng):
    """Rows a quantiser can go wrong at: zeros, one element, both ends equal,
    exact ties, subnormals, NaN and infinity."""
    n, k = w.shape
    tie = hb.f32_to_bf16((np.arange(k) % 16 - 8).astype(np.float32) / 2)
    tie[::32] = 0xC100  # -8: scales of 1, quotients of halves
    one = np.zeros(k, np.uint16)
    one[k // 2] = 0xC123
    ends = np.where(np.arange(k) % 2, 0xBF80, 0x3F80).astype(np.uint16)
    for i, row in enumerate([np.zeros(k, np.uint16), one, ends, tie, rng.integers(0, 40, k).astype(np.uint16)]):
        if i < n:
            w[i] = row
    if n > 6:
        w[5, k // 3], w[6, 0] = 0x7FC1, 0xFF80
    if n > 7:  # the largest finite sizes
        w[7] = np.where(rng.integers(0, 2, k), 0x7F7F, 0xFF7F)
    return w


@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("k,n", SHAPES)
def test_quantize(gpu, k, n, group):
    rng = np.random.default_rng(7 * k + n + group)
    w = special_rows(hb.normal_bf16(k + n, 0.02, (n, k)), rng)
    codes, scales = q4.quantize(w, group)
    a = gpu.alloc_with(np.concatenate([np.zeros(1, np.uint16), w.reshape(-1)]))
    packed = gpu.alloc_with(np.full(hb.q4_bytes(k, n, group) + 16, 0x77, np.uint8))
    good = np.repeat(scales != 0x7FC0, group, axis=1)[:, :k]
    out = gpu.alloc(n * k * 2)
    try:
        run(gpu, hb.q4_quantize(k, n, group), [hb.r(a, 2), hb.r(packed, 0, hb.q4_bytes(k, n, group))], 1)
        run(gpu, hb.q4_dequantize(k, n, group), [hb.r(packed), hb.r(out)], 1)
        got = gpu.download(out, np.uint16, n * k).reshape(n, k)
        tail = gpu.download(packed, np.uint8, 16, hb.q4_bytes(k, n, group))
        # The same bytes as packing the codes themselves.
        w2 = q4.pack(gpu, codes, scales, k, n, group)
        size = hb.q4_bytes(k, n, group)
        same = np.array_equal(gpu.download(w2, np.uint8, size), gpu.download(packed, np.uint8, size))
        gpu.free(w2)
    finally:
        for b in (a, packed, out):
            gpu.free(b)
    assert np.isnan(hb.bf16_to_f32(got[~good])).all()
    want = hb.f32_to_bf16(q4.values(codes, np.where(scales == 0x7FC0, 0, scales), group).astype(np.float32))
    assert np.array_equal(got[good], want[good])
    assert same and (tail == 0x77).all()


# (rows, split, waves, unroll): the defaults, and what a descriptor may name.
FORMS = [(0, 0, 0, 0), (32, 1, 1, 1), (64, 2, 4, 3), (32, 16, 16, 1), (64, 8, 8, 4)]


def matvec(gpu, codes, scales, x, k, n, group, out, mv_m=None, form=(0, 0, 0, 0), y0=None, odd=False):
    m = x.shape[0]
    f32 = out == hb.Out.F32
    nout = n // 2 if out == hb.Out.Swiglu else n
    y0 = np.zeros((m, nout), np.float32 if f32 else np.uint16) if y0 is None else y0
    w = q4.pack(gpu, codes, scales, k, n, group)
    size, pad = y0.dtype.itemsize, 1 if odd else 0
    xb = gpu.alloc_with(np.concatenate([np.full(pad, 0x7FC0, np.uint16), x.reshape(-1), np.full(8, 0x7FC0, np.uint16)]))
    mark = np.full(pad + m * nout + 8, 0x4242, y0.dtype)
    mark[pad:pad + m * nout] = y0.reshape(-1)
    yb = gpu.alloc_with(mark)
    try:
        d = hb.matvec_q4(k, n, out, group, mv_m or m, *form)
        run(gpu, d, [hb.r(w), hb.r(xb, 2 * pad), hb.r(yb, size * pad)], m)
        got = gpu.download(yb, y0.dtype, mark.size)
    finally:
        for b in (w, xb, yb):
            gpu.free(b)
    assert (got[:pad] == mark[:pad]).all() and (got[pad + m * nout:] == mark[pad + m * nout:]).all()
    return got[pad:pad + m * nout].reshape(m, nout)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("k,n,m", [(8, 1, 1), (128, 16, 16), (136, 17, 3), (1000, 33, 2), (2568, 50, 5), (4096, 64, 1),
                                   (1288, 259, 16)])
def test_matvec_exact(gpu, k, n, m, group, form):
    """Small whole x under scales of powers of two: every sum is exact, so the
    f32 outputs equal the definition's."""
    rng = np.random.default_rng(k + n + m + group)
    codes, scales = q4.exact_codes(rng, n, k, group)
    x = hb.f32_to_bf16(rng.integers(-4, 5, (m, k)).astype(np.float32))
    got = matvec(gpu, codes, scales, x, k, n, group, hb.Out.F32, mv_m=min(16, m + m % 2), form=form, odd=True)
    want = hb.bf16_to_f32(x).astype(np.float64) @ q4.values(codes, scales, group).T
    assert np.abs(want).max() < 2 ** 22  # of multiples of 1/4: exact in f32
    assert np.array_equal(got.astype(np.float64), want)


@pytest.mark.parametrize("out", [hb.Out.Bf16, hb.Out.F32, hb.Out.Residual, hb.Out.Swiglu])
@pytest.mark.parametrize("k,n,m,group", [(2560, 96, 1, 32), (5000, 160, 3, 128), (1024, 3584, 16, 64), (17408, 64, 8, 32)])
def test_matvec(gpu, k, n, m, group, out):
    rng = np.random.default_rng(k + n)
    codes, scales = q4.random_codes(rng, n, k, group)
    xf = rng.normal(0, 1, (m, k)) * np.where(rng.random(k) < 0.01, 10, 1)
    x = hb.f32_to_bf16(xf.astype(np.float32))
    xf = hb.bf16_to_f32(x).astype(np.float64)
    y0 = hb.normal_bf16(3, 1.0, (m, n)) if out == hb.Out.Residual else None
    got = matvec(gpu, codes, scales, x, k, n, group, out, y0=y0, odd=out != hb.Out.Swiglu)
    want = xf @ q4.values(codes, scales, group).T
    bound = q4.sum_bound(xf, codes, scales, group)
    if out == hb.Out.Residual:
        want = want + hb.bf16_to_f32(y0)
        bound = bound + q4.U * np.abs(want)
    if out == hb.Out.Swiglu:
        g, u = want[:, :n // 2], want[:, n // 2:]
        bound = q4.swiglu_bound(g, u, bound[:, :n // 2], bound[:, n // 2:])
        want = q4.silu(g) * u
    q4.close(got, want, bound, "matvec_q4")


def test_matvec_non_finite(gpu):
    """A NaN in one row of x makes that row NaN and no other; a NaN scale one
    column; an infinite x gives NaN."""
    k, n, m = 264, 40, 4
    rng = np.random.default_rng(1)
    codes, scales = q4.random_codes(rng, n, k, 64)
    x = hb.normal_bf16(5, 1.0, (m, k))
    clean = matvec(gpu, codes, scales, x, k, n, 64, hb.Out.F32)
    x[1, 263] = 0x7FC0
    x[3, 0] = 0x7F80
    scales[7, 4] = 0x7FC0
    got = matvec(gpu, codes, scales, x, k, n, 64, hb.Out.F32)
    assert np.isnan(got[[1, 3]]).all() and np.isnan(got[:, 7]).all()
    keep = np.arange(n) != 7
    assert np.array_equal(got[0, keep], clean[0, keep]) and np.array_equal(got[2, keep], clean[2, keep])


def test_engine_choice(gpu):
    """Engine.mv_q4: every form it may pick gives the exact sums, the choice
    leaves y as it was, and pins."""
    k, n, m = 1032, 96, 3
    rng = np.random.default_rng(9)
    codes, scales = q4.exact_codes(rng, n, k, 32)
    x = hb.f32_to_bf16(rng.integers(-4, 5, (m, k)).astype(np.float32))
    want = hb.bf16_to_f32(x).astype(np.float64) @ q4.values(codes, scales, 32).T
    w = q4.pack(gpu, codes, scales, k, n, 32)
    xb, y0 = gpu.alloc_with(x), hb.normal_bf16(2, 1.0, (m, n))
    yb, fb = gpu.alloc_with(y0), gpu.alloc(m * n * 4)
    try:
        with hb.Engine(gpu, "") as e:
            for d in e.matvec_q4_candidates(k, n, hb.Out.F32, 32, m):
                run(gpu, d, [hb.r(w), hb.r(xb), hb.r(fb)], m)
                assert np.array_equal(gpu.download(fb, np.float32, m * n).reshape(m, n), want), d
            kern = e.mv_q4(k, n, hb.Out.Residual, 32, m, [hb.r(w)], hb.r(xb), hb.r(yb))
            assert np.array_equal(gpu.download(yb, np.uint16, m * n).reshape(m, n), y0)
            assert e.mv_q4(k, n, hb.Out.Residual, 32, m, [hb.r(w)], hb.r(xb), hb.r(yb)) == kern
            text = e.picks()
            assert text.startswith("mv_q4\t%dx%d q4/32 Residual m%d\t" % (k, n, m))
            with hb.Engine(gpu, "") as e2:
                e2.pin(text)
                assert e2.mv_q4(k, n, hb.Out.Residual, 32, m, [hb.r(w)], hb.r(xb), hb.r(yb)) == kern
        with hb.Engine(gpu, "mv.auto=0") as e:
            assert e.mv_q4(k, n, hb.Out.F32, 32, m, [hb.r(w)], hb.r(xb), hb.r(fb)) == gpu.pipeline(hb.matvec_q4(k, n, hb.Out.F32, 32, m))
    finally:
        for b in (w, xb, yb, fb):
            gpu.free(b)


# ---- the routed experts ----

def route_tables(rng, t, top_k, experts, skew=False):
    """(list, tiles, expert of each sorted pair) of a random route."""
    ids = np.stack([np.sort(rng.choice(experts if not skew else top_k + 1, top_k, replace=False)) for _ in range(t)])
    order = np.argsort(ids.reshape(-1), kind="stable")
    e = ids.reshape(-1)[order]
    table = []
    for x in np.unique(e):
        at = np.flatnonzero(e == x)
        table += [(x, at[0] + o, min(16, len(at) - o)) for o in range(0, len(at), 16)]
    tiles = np.zeros(1 + 3 * hb.moe_tiles(t, top_k, experts, 16), np.uint32)
    tiles[0] = len(table)
    tiles[1:1 + 3 * len(table)] = np.array(table, np.uint32).reshape(-1)
    return order.astype(np.uint32), tiles, e


@pytest.mark.parametrize("t,top_k,experts,h,mi,group,skew", [(1, 8, 64, 256, 64, 32, False), (5, 4, 64, 264, 48, 64, False),
                                                           (40, 4, 16, 512, 112, 128, True), (300, 2, 16, 128, 32, 32, False)])
def test_experts(gpu, t, top_k, experts, h, mi, group, skew):
    rng = np.random.default_rng(t + h)
    lst, tiles, e = route_tables(rng, t, top_k, experts, skew)
    pairs = t * top_k
    gu, gs = q4.random_codes(rng, experts * 2 * mi, h, group)
    dn, ds = q4.exact_codes(rng, experts * h, mi, group)
    wg, wd = q4.pack(gpu, gu, gs, h, 2 * mi, group, experts), q4.pack(gpu, dn, ds, mi, h, group, experts)
    x = hb.normal_bf16(t, 1.0, (t, h))
    hx = hb.f32_to_bf16(rng.integers(-4, 5, (pairs, mi)).astype(np.float32))
    rows_max = t + 3  # kernels of a larger block
    tiles_max = np.zeros(1 + 3 * hb.moe_tiles(rows_max, top_k, experts, 16), np.uint32)
    tiles_max[:tiles.size] = tiles
    bufs = [gpu.alloc_with(a) for a in (np.array([0, 0, 0, t], np.uint32), x, lst, tiles_max, hx)]
    st, xb, lb, tb, hxb = bufs
    hm, ym = np.full(pairs * mi + 64, 0x4242, np.uint16), np.full(pairs * h + 64, 0x4242, np.uint16)
    hb_, yb = gpu.alloc_with(hm), gpu.alloc_with(ym)
    try:
        run(gpu, hb.experts_q4(h, 2 * mi, hb.Out.Swiglu, group, hb.Rows.Gather, top_k, experts, rows_max),
            [hb.r(st), hb.r(wg), hb.r(xb), hb.r(hb_), hb.r(lb), hb.r(tb)], t)
        run(gpu, hb.experts_q4(mi, h, hb.Out.Bf16, group, hb.Rows.Scatter, top_k, experts, rows_max),
            [hb.r(st), hb.r(wd), hb.r(hxb), hb.r(yb), hb.r(lb), hb.r(tb)], t)
        gh, gy = gpu.download(hb_, np.uint16, hm.size), gpu.download(yb, np.uint16, ym.size)
    finally:
        for b in bufs + [wg, wd, hb_, yb]:
            gpu.free(b)
    assert (gh[pairs * mi:] == 0x4242).all() and (gy[pairs * h:] == 0x4242).all()
    gh, gy = gh[:pairs * mi].reshape(pairs, mi), gy[:pairs * h].reshape(pairs, h)
    for ex in np.unique(e):
        p = np.flatnonzero(e == ex)
        c, s = gu[ex * 2 * mi:(ex + 1) * 2 * mi], gs[ex * 2 * mi:(ex + 1) * 2 * mi]
        xf = hb.bf16_to_f32(x[lst[p] // top_k]).astype(np.float64)
        both, eb = xf @ q4.values(c, s, group).T, q4.sum_bound(xf, c, s, group)
        g, u = both[:, :mi], both[:, mi:]
        q4.close(gh[p], q4.silu(g) * u, q4.swiglu_bound(g, u, eb[:, :mi], eb[:, mi:]), "gate|up of expert %d" % ex)
        w = q4.values(dn[ex * h:(ex + 1) * h], ds[ex * h:(ex + 1) * h], group)
        want = hb.bf16_to_f32(hx[p]).astype(np.float64) @ w.T
        assert np.array_equal(gy[lst[p]], hb.f32_to_bf16(want.astype(np.float32))), ex  # exact sums, one rounding


def test_experts_rows_of_state(gpu):
    """state[3] below the launch's rows: tiles past its pairs do nothing."""
    t, top_k, experts, h, mi = 12, 2, 16, 128, 32
    rng = np.random.default_rng(3)
    dn, ds = q4.exact_codes(rng, experts * h, mi, 32)
    wd = q4.pack(gpu, dn, ds, mi, h, 32, experts)
    lst, tiles, e = route_tables(rng, t, top_k, experts)
    hx = hb.f32_to_bf16(rng.integers(-4, 5, (t * top_k, mi)).astype(np.float32))
    mark = np.full(t * top_k * h, 0x4242, np.uint16)
    bufs = [gpu.alloc_with(a) for a in (np.zeros(4, np.uint32), hx, lst, tiles, mark)]
    try:
        k = hb.experts_q4(mi, h, hb.Out.Bf16, 32, hb.Rows.Scatter, top_k, experts, t)
        run(gpu, k, [hb.r(bufs[0]), hb.r(wd), hb.r(bufs[1]), hb.r(bufs[4]), hb.r(bufs[2]), hb.r(bufs[3])], t)
        assert np.array_equal(gpu.download(bufs[4], np.uint16, mark.size), mark)
    finally:
        for b in bufs + [wd]:
            gpu.free(b)


def test_rows_stand_alone(gpu):
    """A row's bits depend neither on the launch's rows nor on the others: in
    the matvec, and for a token of the experts alone and in a batch."""
    k, n = 1032, 80
    rng = np.random.default_rng(11)
    codes, scales = q4.random_codes(rng, n, k, 64)
    x = hb.normal_bf16(8, 1.0, (16, k))
    full = matvec(gpu, codes, scales, x, k, n, 64, hb.Out.F32, mv_m=16)
    for rows in (slice(0, 1), slice(3, 8), slice(5, 16)):
        assert np.array_equal(matvec(gpu, codes, scales, x[rows], k, n, 64, hb.Out.F32, mv_m=16), full[rows])
    t, top_k, experts, h = 30, 2, 16, 96
    dn, ds = q4.random_codes(rng, experts * h, k, 64)
    w = q4.pack(gpu, dn, ds, k, h, 64, experts)
    hx = hb.normal_bf16(9, 1.0, (t * top_k, k))
    kern = hb.experts_q4(k, h, hb.Out.Bf16, 64, hb.Rows.Scatter, top_k, experts, t)

    def down(pairs_x, expert_of):
        """y rows of sorted pairs whose experts are given in order."""
        table = []
        for e in np.unique(expert_of):
            at = np.flatnonzero(expert_of == e)
            table += [(e, at[0] + o, min(16, len(at) - o)) for o in range(0, len(at), 16)]
        tiles = np.zeros(1 + 3 * hb.moe_tiles(t, top_k, experts, 16), np.uint32)
        tiles[0] = len(table)
        tiles[1:1 + 3 * len(table)] = np.array(table, np.uint32).reshape(-1)
        m = len(pairs_x) // top_k
        bufs = [gpu.alloc_with(a) for a in (np.array([0, 0, 0, m], np.uint32), pairs_x, np.zeros(len(pairs_x) * h, np.uint16),
                                            np.arange(len(pairs_x), dtype=np.uint32), tiles)]
        try:
            st, xb, yb, lb, tb = bufs
            run(gpu, kern, [hb.r(st), hb.r(w), hb.r(xb), hb.r(yb), hb.r(lb), hb.r(tb)], m)
            return gpu.download(yb, np.uint16, len(pairs_x) * h).reshape(-1, h)
        finally:
            for b in bufs:
                gpu.free(b)

    batch = down(hx, np.repeat([2, 9, 15], 20))
    for i in (0, 19, 23, 58):
        alone = down(np.concatenate([hx[i:i + 1], hx[i:i + 1]]), np.array([[2, 9, 15][i // 20]] * 2))
        assert np.array_equal(alone[0], batch[i]) and np.array_equal(alone[1], batch[i]), i
    gpu.free(w)
