"""The forms of the 8-bit GEMM that its defaults take, each over shapes that none
of them divides, and outputs at any element of a buffer: exactly where every sum
is exact in f32, and within a bound from its additions elsewhere."""
import numpy as np
import pytest

import f8_ref as f8
import herbert_hip as hb
from test_gpu_f8 import Bufs, marked, quantized_rows, run, same_rows
from test_gpu_f8_gemm import check_h

pytestmark = pytest.mark.gpu


def form(bm, bn, wm, wn, stages, sched):
    return dict(bm=bm, bn=bn, wm=wm, wn=wn, stages=stages, sched=sched)


# What the defaults take by the output (tests/test_f8_host_forms.py holds them to
# these), whole and in parts of K.
DENSE = [form(256, 256, 4, 2, 2, 1), form(128, 160, 4, 2, 2, 1), form(128, 128, 4, 2, 2, 1), form(64, 128, 2, 2, 2, 1), form(32, 64, 1, 4, 3, 0),
         form(32, 32, 1, 2, 4, 0)]
F32 = [form(128, 128, 4, 2, 2, 1), form(64, 128, 2, 4, 2, 0), form(32, 64, 1, 4, 3, 0), form(32, 32, 1, 2, 4, 0)]
SWIGLU = [form(256, 256, 4, 2, 2, 0), form(128, 256, 4, 4, 3, 0), form(64, 256, 2, 4, 3, 0), form(32, 256, 1, 8, 4, 0)]
BY_OUT = [(out, f) for out in (hb.Out.Bf16, hb.Out.Residual) for f in DENSE] + [(hb.Out.F32, f) for f in F32]
EXPERTS = [(32, True), (64, True), (128, True), (32, False), (64, False), (128, False)]  # tile rows, gate and up


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


@pytest.mark.parametrize("parts", [1, 2, 4, 8])
@pytest.mark.parametrize("out,tile", BY_OUT)
@pytest.mark.parametrize("m,k,n", [(1, 1024, 1), (35, 1040, 72), (130, 1184, 333), (515, 2192, 776), (300, 2320, 1026)])
def test_default_forms(gpu, m, k, n, out, tile, parts):
    """One to three K tiles a part, the last one short, rows and columns that no tile divides."""
    exact(gpu, out, m, k, n, **dict(tile, ksplit=parts))


@pytest.mark.parametrize("out,tile", BY_OUT)
@pytest.mark.parametrize("m,k,n", [(1, 16, 1), (129, 128, 258), (257, 272, 136)])
def test_short_k(gpu, m, k, n, out, tile):
    """One or two K tiles, fewer than a form has stages."""
    exact(gpu, out, m, k, n, **tile)


@pytest.mark.parametrize("parts", [1, 4])
@pytest.mark.parametrize("out,tile", BY_OUT)
def test_default_forms_random(gpu, out, tile, parts):
    """Weights as a model's are, against 64 bits."""
    rng = np.random.default_rng(parts + tile["bm"])
    m, k, n = 290, 2064, 664
    codes, scales = f8.random_weights(rng, n, k)
    x = hb.normal_bf16(parts, 1.0, (m, k))
    xv, wv = f8.row_values(*f8.quantize_rows(x)), f8.values(codes, scales)
    want, bound = xv @ wv.T, (f8.sum_bound if out == hb.Out.F32 else f8.mfma_bound)(xv, wv)
    y0 = hb.normal_bf16(7, 1.0, (m, n)) if out != hb.Out.F32 else np.zeros((m, n), np.float32)
    if out == hb.Out.Residual:
        want = want + f8.f64(y0)
        bound = bound + f8.U * np.abs(want)
    f8.close(gemm(gpu, codes, scales, x, out, y0, **dict(tile, ksplit=parts)), want, bound, "gemm_f8")


def swiglu_close(raw, m, n, s, bound=0.0):
    g, u = s[:, :n], s[:, n:]
    eg, eu = (bound[:, :n], bound[:, n:]) if np.ndim(bound) else (bound, bound)
    check_h(raw, m, n, f8.silu(g) * u, f8.swiglu_bound(g, u, eg, eu))


@pytest.mark.parametrize("tile", SWIGLU)
@pytest.mark.parametrize("m,k,n", [(1, 16, 256), (35, 144, 512), (300, 400, 768), (515, 1184, 256)])
def test_default_swiglu(gpu, tile, m, k, n):
    rng = np.random.default_rng(m + k + n)
    codes, scales = f8.exact_weights(rng, n, k)
    scales = scales * np.float32(2.0 ** -10)  # sums around 1
    x = f8.exact_x(rng, m, k)
    raw = gemm(gpu, codes, scales, x, hb.Out.Swiglu, marked((m, hb.f8_row_bytes(n // 2))), **tile)
    swiglu_close(raw, m, n // 2, f8.f64(x) @ f8.values(codes, scales).T)


@pytest.mark.parametrize("bm,gate_up", EXPERTS)
def test_default_experts(gpu, bm, gate_up):
    """The experts' products in the forms that experts_f8 leaves to the defaults, over tiles full, short
    and of one row."""
    k, n, top_k = 400, 512, 2
    rng = np.random.default_rng(bm + gate_up)
    counts = [bm, 2 * bm + 1, 0, 5, 2 * bm - 6]
    pairs, experts = sum(counts), len(counts)
    t = pairs // top_k
    w = [f8.exact_weights(rng, n, k) for _ in range(experts)]
    w = [(c, s * np.float32(2.0 ** -10 if gate_up else 1.0)) for c, s in w]
    order = rng.permutation(pairs).astype(np.uint32)
    tab, first = [], 0
    for e, count in enumerate(counts):
        tab += [(e, first + i, min(bm, count - i)) for i in range(0, count, bm)]
        first += count
    tiles = np.zeros(1 + 3 * hb.moe_tiles(t, top_k, experts, bm), np.uint32)
    tiles[0] = len(tab)
    tiles[1:1 + 3 * len(tab)] = np.array(tab, np.uint32).reshape(-1)
    x = f8.exact_x(rng, t if gate_up else pairs, k)
    y0 = marked((pairs, hb.f8_row_bytes(n // 2))) if gate_up else np.full((pairs, n), 0x4242, np.uint16)
    out, rows = (hb.Out.Swiglu, hb.Rows.Gather) if gate_up else (hb.Out.Bf16, hb.Rows.Scatter)
    with Bufs(gpu) as b:
        st, ls, tl, wr = b.put(np.array([0, 0, 0, t], np.uint32)), b.put(order), b.put(tiles), b.put(np.concatenate([f8.pack(*v) for v in w]))
        xr, y = b.put(f8.pack_rows(*f8.quantize_rows(x))), b.put(y0)
        run(gpu, hb.experts_f8(k, n, out, rows, top_k, experts, t, bm), [st, wr, xr, y, ls, tl], t)
        got = b.get(y, y0.dtype, y0.shape)
    expert = np.repeat(np.arange(experts), counts)
    xv = f8.f64(x)
    for p in range(pairs):
        row = xv[order[p] // top_k] if gate_up else xv[p]
        want = (row @ f8.values(*w[expert[p]]).T)[None]
        if gate_up:
            swiglu_close(got[p:p + 1], 1, n // 2, want)
        else:
            np.testing.assert_array_equal(got[order[p]], hb.f32_to_bf16(want.astype(np.float32))[0])


def quotient_rows():
    """bf16 rows of groups of 128, each its largest, t, beside 127 others, so that every x below or
    equal to it stands beside it at every distance of their exponents: at each, t twice, the first
    group without the last x, the second without the first, the one the largest's place."""
    rows = []
    for d in range(24):
        x = (0x3F80 - (d << 7) + np.arange(128)).astype(np.uint16)  # 2^-d .. 2^(1-d)
        for t in (0x3F80 + np.arange(128)).astype(np.uint16):
            for at in (127, 0):
                g = np.where(x > t, np.uint16(0), x)
                g[at] = t
                rows.append(g)
    return np.array(rows, np.uint16)


def test_every_quotient_beside_its_largest(gpu):
    groups = quotient_rows()
    top = groups.max(1)
    seen = np.zeros((24, 128, 128), bool)  # distance, mantissa of the largest, of the other
    for d in range(24):
        part = groups[256 * d:256 * (d + 1)]
        in_range = part >> 7 == 127 - d
        seen[d, np.repeat(top[256 * d:256 * (d + 1)] & 127, 128)[in_range.ravel()], (part & 127)[in_range]] = True
    assert (top >> 7 == 127).all() and seen[1:].all()
    below = np.arange(128)[:, None] >= np.arange(128)[None, :]
    assert (seen[0] == below).all()
    x = groups.reshape(-1, 128 * 16)
    x[1::2] ^= 0x8000
    same_rows(*quantized_rows(gpu, x), x)
