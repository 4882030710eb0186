"""The forms of matvec_q4 that a shape's defaults, the engine or a descriptor
name: 16 to 128 W rows a wave, K shared by 1 to 16 waves, every number of x
rows, over one matrix and over experts.  Codes under scales of powers of two and
small whole x: every sum is exact in f32 in any order, so all forms have the
same sums, the definition's in 64 bits."""
import numpy as np
import pytest

import herbert_hip as hb
import q4_ref as q4

pytestmark = pytest.mark.gpu

GROUP = 64


def small_codes(rng, n, k, group=GROUP):
    """q4.exact_codes with sums of about 1, where the SwiGLU is no straight
    line: whole multiples of 2^-12, below 2^9."""
    codes, scales = q4.exact_codes(rng, n, k, group)
    return codes, hb.f32_to_bf16(hb.bf16_to_f32(scales) * np.float32(2.0 ** -10))


def whole_x(rng, m, k):
    return hb.f32_to_bf16(rng.integers(-4, 5, (m, k)).astype(np.float32))


def sums(x, codes, scales, group=GROUP):
    """x . W^T in 64 bits, parts of W at a time."""
    xf = hb.bf16_to_f32(x).astype(np.float64)
    y = np.concatenate([xf @ q4.values(codes[i:i + 4096], scales[i:i + 4096], group).T for i in range(0, len(codes), 4096)], 1)
    # What makes an f32 sum exact: multiples of 2^-12 that 24 bits hold.
    assert np.array_equal(y * 4096, np.rint(y * 4096)) and np.abs(y).max() < 512
    return y


def check(got, y, out, what):
    """Outputs of the exact sums y: equal where Out rounds once, within the
    arithmetic of the SwiGLU.  (Gates here are below 8 in size: e^-g is off by
    8 + 2 half steps of f32 at most, the division, the sum and the two products
    by half a step each, of the 16 whole steps that swiglu_bound has.)"""
    if out == hb.Out.F32:
        assert np.array_equal(got, y.astype(np.float32)), what
    elif out == hb.Out.Bf16:
        assert np.array_equal(got, hb.f32_to_bf16(y.astype(np.float32))), what
    else:
        half = y.shape[1] // 2
        g, u = y[:, :half], y[:, half:]
        assert not g.size or np.abs(g).max() < 8
        q4.close(got, q4.silu(g) * u, q4.swiglu_bound(g, u, 0.0, 0.0), what)


class Matrix:
    """A packed matrix with its x rows and the sums of 16 of them."""

    def __init__(self, gpu, k, n, seed):
        rng = np.random.default_rng(seed)
        codes, scales = small_codes(rng, n, k)
        self.gpu, self.k, self.n = gpu, k, n
        self.x = whole_x(rng, 16, k)
        self.y = sums(self.x, codes, scales)
        self.w, self.xb = q4.pack(gpu, codes, scales, k, n, GROUP), gpu.alloc_with(self.x)
        self.yb = gpu.alloc(16 * n * 4 + 64)

    def free(self):
        for b in (self.w, self.xb, self.yb):
            self.gpu.free(b)

    def run(self, d, m):
        """The outputs of a launch over m rows, nothing written past them."""
        gpu = self.gpu
        kind = np.float32 if d.out == hb.Out.F32 else np.uint16
        count = m * (self.n // 2 if d.out == hb.Out.Swiglu else self.n)
        gpu.upload(self.yb, np.full(count + 16, 0x4242, kind))
        kern = gpu.pipeline(d)
        gpu.launch(kern, [hb.r(self.w), hb.r(self.xb), hb.r(self.yb)], m)
        got = gpu.download(self.yb, kind, count + 16)
        assert (got[count:] == np.full(1, 0x4242, kind)).all(), gpu.kernel_name(kern)
        check(got[:count].reshape(m, -1), self.y[:m], d.out, gpu.kernel_name(kern))


def form(d):
    return (d.rows, d.split, d.mv_waves, d.unroll)


@pytest.fixture(scope="module")
def wide(gpu):
    """Where the engine has every row width to choose from, and K for sixteen waves."""
    m = Matrix(gpu, 2056, 16416, 31)
    yield m
    m.free()


@pytest.mark.parametrize("out", [hb.Out.F32, hb.Out.Swiglu])
@pytest.mark.parametrize("m", [1, 4, 8, 16])
def test_engine_candidates(gpu, wide, m, out):
    with hb.Engine(gpu, "") as e:
        descs = e.matvec_q4_candidates(wide.k, wide.n, out, GROUP, m)
    assert {d.rows for d in descs} == ({16, 32, 64, 128} if out == hb.Out.F32 else {32, 64, 128})
    assert {d.split for d in descs} == {4, 8, 16}
    for d in descs:
        wide.run(d, m)


@pytest.fixture(scope="module")
def narrow(gpu):
    m = Matrix(gpu, 1032, 416, 32)
    yield m
    m.free()


@pytest.mark.parametrize("out", [hb.Out.F32, hb.Out.Swiglu])
@pytest.mark.parametrize("rows,split,waves,unroll", [(32, 1, 4, 2), (64, 1, 1, 1), (64, 2, 8, 1), (64, 16, 16, 1), (128, 1, 2, 1),
                                                     (128, 4, 4, 1), (128, 8, 16, 1)])
def test_forms_by_rows(gpu, narrow, rows, split, waves, unroll, out):
    """Each way that a wave's quads share its row tiles, at 1 to 16 x rows."""
    for m in (1, 3, 4, 6, 8, 11, 16):
        narrow.run(hb.matvec_q4(narrow.k, narrow.n, out, GROUP, m, rows, split, waves, unroll), m)


@pytest.mark.parametrize("n,m,rows", [(65568, 9, 128), (65568, 16, 128), (65568, 8, 64), (65536, 16, 32), (4128, 3, 32), (4096, 3, 16)])
def test_defaults(gpu, n, m, rows):
    """The defaults on both sides of each of their borders."""
    mat = Matrix(gpu, 264, n, n + m)
    try:
        for out in (hb.Out.F32, hb.Out.Bf16, hb.Out.Swiglu):
            d = hb.matvec_q4(264, n, out, GROUP, m)
            assert "_r%d_" % max(rows, 32 if out == hb.Out.Swiglu else 16) in gpu.kernel_name(gpu.pipeline(d))
            mat.run(d, m)
    finally:
        mat.free()


# ---- over experts ----

class Experts:
    """A block of t rows routed to some experts, some with several tiles of 16
    rows, some with a few and some with no row."""

    def __init__(self, gpu, t, top_k, experts, h, n, seed):
        rng = np.random.default_rng(seed)
        self.gpu, self.t, self.top_k, self.experts, self.h, self.n = gpu, t, top_k, experts, h, n
        codes, scales = small_codes(rng, experts * n, h)
        pairs = t * top_k
        # A third of the rows to the same experts.
        ids = np.stack([np.arange(top_k) if i % 3 == 0 else np.sort(rng.choice(experts - 1, top_k, replace=False)) for i in range(t)])
        self.list = np.argsort(ids.reshape(-1), kind="stable").astype(np.uint32)
        self.e = ids.reshape(-1)[self.list]
        self.table = []
        for x in np.unique(self.e):
            at = np.flatnonzero(self.e == x)
            self.table += [(x, at[0] + o, min(16, len(at) - o)) for o in range(0, len(at), 16)]
        self.x, self.sorted_x = whole_x(rng, t, h), whole_x(rng, pairs, h)
        self.y = {}
        for rows_of, xr in ((hb.Rows.Gather, self.x[self.list // top_k]), (hb.Rows.Scatter, self.sorted_x)):
            y = np.empty((pairs, n))
            for x in np.unique(self.e):
                at = np.flatnonzero(self.e == x)
                y[at] = sums(xr[at], codes[x * n:(x + 1) * n], scales[x * n:(x + 1) * n])
            self.y[rows_of] = y
        self.w = q4.pack(gpu, codes, scales, h, n, GROUP, experts)
        self.bufs = [gpu.alloc_with(a) for a in (self.x, self.sorted_x, self.list)]

    def free(self):
        for b in self.bufs + [self.w]:
            self.gpu.free(b)

    def run(self, rows_of, out, rows_max, state=None, **fields):
        """A launch over the block, with state[3] = `state` rows of it: (name,
        outputs, which rows they may be in).  The rest stays as it was."""
        gpu, pairs = self.gpu, self.t * self.top_k
        width = self.n // 2 if out == hb.Out.Swiglu else self.n
        tiles = np.zeros(1 + 3 * hb.moe_tiles(rows_max, self.top_k, self.experts, 16), np.uint32)
        tiles[0] = len(self.table)
        tiles[1:1 + 3 * len(self.table)] = np.array(self.table, np.uint32).reshape(-1)
        kern = gpu.pipeline(hb.experts_q4(self.h, self.n, out, GROUP, rows_of, self.top_k, self.experts, rows_max, **fields))
        x, sx, lst = self.bufs
        mark = np.full(pairs * width + 32, 0x4242, np.uint16)
        tmp = [gpu.alloc_with(a) for a in (np.array([0, 0, 0, self.t if state is None else state], np.uint32), tiles, mark)]
        try:
            bind = [hb.r(tmp[0]), hb.r(self.w), hb.r(x if rows_of == hb.Rows.Gather else sx), hb.r(tmp[2]), hb.r(lst), hb.r(tmp[1])]
            gpu.launch(kern, bind, self.t)
            got = gpu.download(tmp[2], np.uint16, mark.size)
            gpu.upload(tmp[2], mark)
            gpu.launch(kern, bind, self.t)
            assert np.array_equal(gpu.download(tmp[2], np.uint16, mark.size), got), "a second launch's bits"
        finally:
            for b in tmp:
                gpu.free(b)
        name = gpu.kernel_name(kern)
        valid = pairs if state is None else state * self.top_k
        at = np.arange(valid) if rows_of == hb.Rows.Gather else self.list[:valid]
        rest = np.ones(got.size, bool)
        rest[:pairs * width].reshape(pairs, width)[at] = False
        assert (got[rest] == 0x4242).all(), name
        check(got[:pairs * width].reshape(pairs, width)[at], self.y[rows_of][:valid], out, name)
        return name


@pytest.fixture(scope="module")
def routed(gpu):
    x = Experts(gpu, 50, 4, 24, 1032, 224, 41)
    yield x
    x.free()


@pytest.mark.parametrize("rows_of,out", [(hb.Rows.Gather, hb.Out.Swiglu), (hb.Rows.Gather, hb.Out.Bf16), (hb.Rows.Scatter, hb.Out.Bf16)])
@pytest.mark.parametrize("rows,split,waves,unroll", [(32, 8, 0, 2), (64, 1, 1, 1), (64, 4, 4, 1), (64, 16, 0, 1), (128, 1, 4, 1),
                                                     (128, 4, 8, 1), (128, 8, 8, 1)])
def test_expert_forms(routed, rows, split, waves, unroll, rows_of, out):
    name = routed.run(rows_of, out, routed.t + 1, rows=rows, split=split, waves=waves, unroll=unroll)
    assert "_r%d_k%d_" % (rows, split) in name


@pytest.mark.parametrize("rows_of,out", [(hb.Rows.Gather, hb.Out.Swiglu), (hb.Rows.Scatter, hb.Out.Bf16)])
@pytest.mark.parametrize("rows_max,rows", [(50, 32), (2048, 64)])
def test_expert_defaults(routed, rows_max, rows, rows_of, out):
    """Of a small block, and of one whose pairs make 8192 workgroups."""
    assert "_r%d_" % rows in routed.run(rows_of, out, rows_max)


@pytest.mark.parametrize("rows_of,out", [(hb.Rows.Gather, hb.Out.Swiglu), (hb.Rows.Gather, hb.Out.Bf16), (hb.Rows.Scatter, hb.Out.Bf16)])
def test_expert_tiles_past_the_rows_of_state(gpu, rows_of, out):
    """state[3] = 5 of a launch over 12 rows, 2 slots: a tile whose 9 rows cross
    the tenth pair runs 3 of them, a tile past it none."""
    x = Experts(gpu, 12, 2, 8, 264, 96, 43)
    try:
        rng = np.random.default_rng(44)
        # The first 10 sorted pairs are the 5 rows' own, in some order.
        x.list = np.concatenate([rng.permutation(10), 10 + rng.permutation(14)]).astype(np.uint32)
        x.table = [(0, 0, 7), (3, 7, 9), (5, 16, 8)]
        expert = np.repeat([0, 3, 5], [7, 9, 8])
        codes, scales = small_codes(np.random.default_rng(45), x.experts * x.n, x.h)
        gpu.free(x.w)
        x.w = q4.pack(gpu, codes, scales, x.h, x.n, GROUP, x.experts)
        gpu.upload(x.bufs[2], x.list)
        for rows, xr in ((hb.Rows.Gather, x.x[x.list // 2]), (hb.Rows.Scatter, x.sorted_x)):
            x.y[rows] = np.concatenate([sums(xr[i:i + 1], codes[e * x.n:(e + 1) * x.n], scales[e * x.n:(e + 1) * x.n])
                                        for i, e in enumerate(expert)])
        for state in (5, 12, 1, 0):
            if state == 1:  # the first pairs are then row 0's
                x.list[:2], x.list[2:10] = (1, 0), 2 + rng.permutation(8)
                gpu.upload(x.bufs[2], x.list)
                xr = x.x[x.list // 2]
                x.y[hb.Rows.Gather] = np.concatenate([sums(xr[i:i + 1], codes[e * x.n:(e + 1) * x.n], scales[e * x.n:(e + 1) * x.n])
                                                      for i, e in enumerate(expert)])
            for rows in (32, 64):
                x.run(rows_of, out, 12, state=state, rows=rows)
    finally:
        x.free()
