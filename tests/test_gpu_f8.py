"""8-bit rows and matrices on the GPU: quantised and read back bit for bit, and
the matvec over an 8-bit matrix, exactly where every sum is exact in f32 and
within a bound from its additions elsewhere."""
import numpy as np
import pytest

import f8_ref as f8
import herbert_hip as hb

pytestmark = pytest.mark.gpu


class Bufs:
    """Buffers freed together."""

    def __init__(self, gpu):
        self.gpu, self.ids = gpu, []

    def put(self, a, odd=0):
        """The array at an offset of `odd` elements, with room marked behind it."""
        a = np.ascontiguousarray(a)
        raw = np.full(odd * a.itemsize + a.nbytes + 64, 0xA5, np.uint8)
        raw[odd * a.itemsize:odd * a.itemsize + a.nbytes] = a.reshape(-1).view(np.uint8)
        self.ids.append(self.gpu.alloc_with(raw))
        return hb.r(self.ids[-1], odd * a.itemsize)

    def get(self, r, dtype, shape):
        n = int(np.prod(shape))
        size = n * np.dtype(dtype).itemsize
        raw = self.gpu.download(r.buf, np.uint8, r.offset + size + 64)
        assert (raw[:r.offset] == 0xA5).all() and (raw[-64:] == 0xA5).all(), "written outside"
        return raw[r.offset:r.offset + size].view(dtype).reshape(shape)

    def __enter__(self):
        return self

    def __exit__(self, *a):
        for b in self.ids:
            self.gpu.free(b)


def marked(shape, dtype=np.uint8):
    return np.full(shape, 0xA5 if dtype == np.uint8 else 0x5A5A, dtype)


def run(gpu, desc, ranges, m):
    gpu.launch(gpu.pipeline(desc), ranges, m)
    gpu.sync()


def quantized_rows(gpu, x, odd=0):
    """The f8 rows of bf16 bits x by the library, and back as bf16."""
    m, k = x.shape
    with Bufs(gpu) as b:
        xr, q = b.put(x, odd), b.put(marked((m, hb.f8_row_bytes(k))))
        back = b.put(marked((m, k), np.uint16), odd)
        run(gpu, hb.f8_quantize_rows(k), [xr, q], m)
        run(gpu, hb.f8_dequantize_rows(k), [q, back], m)
        return b.get(q, np.uint8, (m, hb.f8_row_bytes(k))), b.get(back, np.uint16, (m, k))


def same_rows(raw, back, x):
    m, k = x.shape
    codes, scales = f8.unpack_rows(raw, m, k)
    want, ws = f8.quantize_rows(x)
    bad = ~np.isfinite(ws)
    assert np.array_equal(np.isfinite(scales), ~bad)
    assert np.array_equal(scales[~bad], ws[~bad])
    wide = np.repeat(bad, 128, 1)[:, :k]
    assert np.array_equal(codes[~wide], want[~wide])
    v = f8.f64(back)
    assert np.isnan(v[wide]).all()
    with np.errstate(invalid="ignore"):
        value = f8.VALUES[codes].astype(np.float32) * np.repeat(scales, 128, 1)[:, :k]
    assert np.array_equal(back[~wide], hb.f32_to_bf16(value)[~wide])


@pytest.mark.parametrize("m,k", [(1, 16), (1, 2560), (3, 112), (5, 128), (7, 144), (57, 5008), (33, 1040), (300, 256)])
@pytest.mark.parametrize("odd", [0, 3])
def test_rows(gpu, m, k, odd):
    x = hb.normal_bf16(m * 7 + k, 3.0, (m, k))
    same_rows(*quantized_rows(gpu, x, odd), x)


def test_every_quotient(gpu):
    """Every 8-bit x under every 8-bit largest, at 24 distances of their
    exponents: the ties among them as the definition has them."""
    top = 0x3F80 + np.arange(128)  # 1 .. 2
    rows = []
    for d in range(24):
        x = (0x3F80 - (d << 7) + np.arange(128)).astype(np.uint16)
        for t in top:
            g = np.where(x > t, np.uint16(0), x)
            g[np.argmax(g == 0) if (g == 0).any() else 127] = t
            rows.append(g)
    x = np.array(rows, np.uint16).reshape(-1, 128 * 16)
    x[1::2] ^= 0x8000
    same_rows(*quantized_rows(gpu, x), x)


def test_special_rows(gpu):
    """Groups of zeros, below the smallest scale, subnormal, huge, with an
    infinity or a NaN, beside ordinary ones."""
    x = hb.normal_bf16(5, 1.0, (10, 384))
    x[0, 128:256] = 0
    x[1, 128:256] = hb.f32_to_bf16(np.float32(2.0 ** -104) * hb.bf16_to_f32(x[1, 128:256]))
    x[2, 128:256] = np.arange(128)  # subnormals
    x[3, :128] = hb.f32_to_bf16(np.float32(2.0 ** 125) * np.clip(hb.bf16_to_f32(x[3, :128]), -3, 3))
    x[4, 5] = 0x7F80
    x[5, 200] = 0xFF80
    x[6, 383] = 0x7FC0
    x[7, 0] = 0xFFFF
    x[8, 128:256] = 0x8000
    x[9, 1] = 0x7F7F  # the largest
    same_rows(*quantized_rows(gpu, x), x)


@pytest.mark.parametrize("n,k,count", [(1, 16, 1), (128, 128, 1), (129, 144, 2), (1000, 640, 1), (300, 5008, 3)])
def test_matrix(gpu, n, k, count):
    w = hb.normal_bf16(n + k, 0.02, (count, n, k))
    w[0, 0, :16] = 0
    size = hb.f8_bytes(k, n)
    with Bufs(gpu) as b:
        wr, q, back = b.put(w, 1), b.put(marked((count, size))), b.put(marked((count, n, k), np.uint16), 1)
        run(gpu, hb.f8_quantize(k, n), [wr, q], count)
        run(gpu, hb.f8_dequantize(k, n), [q, back], count)
        raw, got = b.get(q, np.uint8, (count, size)), b.get(back, np.uint16, (count, n, k))
    for i in range(count):
        codes, scales = f8.quantize(w[i])
        assert np.array_equal(raw[i, :n * k].reshape(n, k), codes)
        assert np.array_equal(raw[i, n * k:n * k + 4 * scales.size].view(np.float32).reshape(scales.shape), scales)
        s = np.repeat(np.repeat(scales, 128, 0)[:n], 128, 1)[:, :k]
        assert np.array_equal(got[i], hb.f32_to_bf16(f8.VALUES[codes].astype(np.float32) * s))


# ---- the matvec ----

def matvec(gpu, codes, scales, x, out, y0=None, odd=0, **form):
    m, k = x.shape
    n = codes.shape[0]
    width = n // 2 if out == hb.Out.Swiglu else n
    dtype = np.float32 if out == hb.Out.F32 else np.uint16
    y = np.full((m, width), 0x42, dtype) if y0 is None else y0
    with Bufs(gpu) as b:
        w, xr, yr = b.put(f8.pack(codes, scales)), b.put(x, 8 * odd), b.put(y, odd)
        run(gpu, hb.matvec_f8(k, n, out, **form), [w, xr, yr], m)
        return b.get(yr, dtype, (m, width))


def check_matvec(gpu, codes, scales, x, out, odd=0, seed=0, **form):
    n = codes.shape[0]
    xv, wv = f8.row_values(*f8.quantize_rows(x)), f8.values(codes, scales)
    want, bound = xv @ wv.T, f8.sum_bound(xv, wv)
    y0 = hb.normal_bf16(seed + 9, 1.0, want.shape) if out == hb.Out.Residual else None
    got = matvec(gpu, codes, scales, x, out, y0, odd, **form)
    if out == hb.Out.Residual:
        want = want + f8.f64(y0)
        bound = bound + f8.U * np.abs(want)
    if out == hb.Out.Swiglu:
        g, u, eg, eu = want[:, :n // 2], want[:, n // 2:], bound[:, :n // 2], bound[:, n // 2:]
        want, bound = f8.silu(g) * u, f8.swiglu_bound(g, u, eg, eu)
    f8.close(got, want, bound, "matvec")


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 8, 13, 16])
@pytest.mark.parametrize("k,n", [(16, 1), (128, 16), (144, 33), (2560, 300), (5008, 130)])
def test_matvec_exact(gpu, m, k, n):
    rng = np.random.default_rng(m * 1000 + k + n)
    codes, scales = f8.exact_weights(rng, n, k)
    x = f8.exact_x(rng, m, k)
    want = f8.row_values(*f8.quantize_rows(x)) @ f8.values(codes, scales).T
    assert np.array_equal(want, f8.f64(x) @ f8.values(codes, scales).T) and np.abs(want).max() * 16 < 2 ** 24
    got = matvec(gpu, codes, scales, x, hb.Out.F32, mv_m=m, odd=m % 2)
    assert np.array_equal(got.astype(np.float64), want)


@pytest.mark.parametrize("m,k,n", [(1, 1152, 40), (4, 400, 70), (16, 1024, 256)])
def test_matvec_wide_products(gpu, m, k, n):
    """Products far apart in size: the small ones stay in the sums."""
    rng = np.random.default_rng(m + n)
    codes, scales = f8.wide_weights(rng, n, k)
    x = f8.exact_x(rng, m, k, (0, 1))
    want = f8.f64(x) @ f8.values(codes, scales).T
    assert np.array_equal(matvec(gpu, codes, scales, x, hb.Out.F32, mv_m=m).astype(np.float64), want)


@pytest.mark.parametrize("rows,split,waves,unroll", [(16, 1, 1, 1), (16, 16, 16, 1), (32, 8, 8, 1), (64, 4, 4, 1), (32, 2, 4, 4),
                                                     (64, 1, 2, 2), (16, 4, 8, 2), (64, 8, 8, 1)])
@pytest.mark.parametrize("out", list(hb.Out))
def test_matvec_forms(gpu, rows, split, waves, unroll, out):
    if out == hb.Out.Swiglu and rows == 16:
        pytest.skip("a wave of the SwiGLU holds a gate and an up tile")
    for m, k, n in [(1, 2048, 512), (3, 2064, 768), (16, 2128, 512 if out == hb.Out.Swiglu else 777), (9, 4096, 256)]:
        rng = np.random.default_rng(rows + split + m)
        codes, scales = f8.random_weights(rng, n, k)
        check_matvec(gpu, codes, scales, hb.normal_bf16(m + k, 1.0, (m, k)), out, odd=1, mv_m=m, rows=rows, split=split, waves=waves,
                     unroll=unroll)


@pytest.mark.parametrize("k,n,m,out", [(2560, 18432, 1, hb.Out.Swiglu), (4096, 2560, 1, hb.Out.Bf16), (9216, 2560, 4, hb.Out.Residual),
                                       (17408, 640, 16, hb.Out.F32), (2560, 70000, 2, hb.Out.F32)])
def test_matvec_defaults(gpu, k, n, m, out):
    rng = np.random.default_rng(k + n)
    codes, scales = f8.random_weights(rng, n, k)
    check_matvec(gpu, codes, scales, hb.normal_bf16(m + k, 1.0, (m, k)), out, mv_m=m)


def test_matvec_rows_apart(gpu):
    """A row's bits depend neither on the launch's rows nor on the others, and a
    row with a NaN or an infinity leaves the others alone."""
    rng = np.random.default_rng(3)
    k, n = 2064, 272
    codes, scales = f8.random_weights(rng, n, k)
    x = hb.normal_bf16(4, 1.0, (16, k))
    kw = dict(out=hb.Out.F32, mv_m=16)
    whole = matvec(gpu, codes, scales, x, **kw)
    for i in (0, 7, 15):
        assert np.array_equal(matvec(gpu, codes, scales, x[i:i + 1], **kw)[0], whole[i])
    x[5, 77], x[9, 2063], x[12] = 0x7FC0, 0x7F80, 0
    got = matvec(gpu, codes, scales, x, **kw)
    assert np.isnan(got[5]).all() and np.isnan(got[9]).all() and (got[12] == 0).all()
    rest = [i for i in range(16) if i not in (5, 9, 12)]
    assert np.array_equal(got[rest], whole[rest])
    codes[100, 3] = 0x7F
    got = matvec(gpu, codes, scales, x, **kw)
    assert np.isnan(got[:, 100]).all() and np.isfinite(got[0, np.arange(n) != 100]).all()
