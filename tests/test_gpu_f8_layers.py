"""The router and the 8-bit operators as they are used together: a decode
layer's projections (eager, and recorded into a graph beside eager work), the
MoE layer and block over 8-bit experts behind either route, a prompt's MLP from
a checkpoint, two contexts at once, a matrix past 4 GiB, and the native host."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import f8_ref as f8
import herbert_hip as hb
import hb_oracle as orc
from route_ref import route as route_ref
from test_gpu_f8_gemm import check_h
from test_zz_no_alloc import run_static

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def packed(gpu, mats):
    """The f8 matrices, one after the other, on the GPU."""
    return gpu.alloc_with(np.concatenate([f8.pack(*w) for w in mats]))


def swiglu_of(xv, w, sums):
    """h = silu(g) u of 8-bit x values, and what it may be off by before it is rounded."""
    wv = f8.values(*w)
    both, eb = xv @ wv.T, sums(xv, wv)
    n = both.shape[1] // 2
    g, u = both[:, :n], both[:, n:]
    return f8.silu(g) * u, f8.swiglu_bound(g, u, eb[:, :n], eb[:, n:])


class Mlp:
    """rows of x through gate|up and down over 8-bit weights: as a decode step's
    two matvecs, or as a prompt's (x quantised, f8 rows of h, x updated)."""

    def __init__(self, gpu, m, h, inter, seed, prompt):
        rng = np.random.default_rng(seed)
        self.gpu, self.m, self.h, self.inter, self.prompt = gpu, m, h, inter, prompt
        self.gu, self.dn = f8.random_weights(rng, 2 * inter, h), f8.random_weights(rng, h, inter)
        hrow = hb.f8_row_bytes(inter) if prompt else 2 * inter
        self.b = {"gu": packed(gpu, [self.gu]), "dn": packed(gpu, [self.dn]), "x": gpu.alloc(m * h * 2), "y": gpu.alloc(m * h * 2),
                  "x8": gpu.alloc(m * hb.f8_row_bytes(h)), "h": gpu.alloc(m * hrow), "state": gpu.alloc_with(np.array([0, 0, 0, m], np.uint32))}
        b = {n: hb.r(v) for n, v in self.b.items()}
        if prompt:
            steps = [(hb.f8_quantize_rows(h), ["x", "x8"]), (hb.gemm_f8(h, 2 * inter, hb.Out.Swiglu, rows=m), ["state", "gu", "x8", "h", "state", "state"]),
                     (hb.gemm_f8(inter, h, hb.Out.Residual, rows=m, ksplit=2), ["state", "dn", "h", "y", "state", "state"])]
        else:
            steps = [(hb.matvec_f8(h, 2 * inter, hb.Out.Swiglu, mv_m=m), ["gu", "x", "h"]), (hb.matvec_f8(inter, h, hb.Out.Residual, mv_m=m), ["dn", "h", "y"])]
        self.steps = [(gpu.pipeline(d), [b[n] for n in names], m) for d, names in steps]

    def feed(self, seed):
        self.x, self.y0 = hb.normal_bf16(seed, 1.0, (self.m, self.h)), hb.normal_bf16(seed + 1, 1.0, (self.m, self.h))
        self.gpu.upload(self.b["x"], self.x)
        self.gpu.upload(self.b["y"], self.y0)

    def launch(self):
        for k, ranges, m in self.steps:
            self.gpu.launch(k, ranges, m)

    def results(self):
        self.gpu.sync()
        return (self.gpu.download(self.b["h"], np.uint8, self.gpu.size(self.b["h"])).reshape(self.m, -1),
                self.gpu.download(self.b["y"], np.uint16, self.m * self.h).reshape(self.m, self.h))

    def check(self):
        h, y = self.results()
        sums = f8.mfma_bound if self.prompt else f8.sum_bound
        want, bound = swiglu_of(f8.row_values(*f8.quantize_rows(self.x)), self.gu, sums)
        if self.prompt:
            check_h(h, self.m, self.inter, want, bound)
            hv = f8.row_values(*f8.unpack_rows(h, self.m, self.inter))
        else:
            bits = h.reshape(-1).view(np.uint16).reshape(self.m, self.inter)
            f8.close(bits, want, bound, "h")
            hv = f8.row_values(*f8.quantize_rows(bits))
        wv = f8.values(*self.dn)
        want = hv @ wv.T + f8.f64(self.y0)
        f8.close(y, want, sums(hv, wv) + f8.U * np.abs(want), "y")

    def free(self):
        for b in self.b.values():
            self.gpu.free(b)


FORMS = [(1, False), (5, False), (16, False), (70, True)]


@pytest.mark.parametrize("m,prompt", FORMS)
def test_mlp(gpu, m, prompt):
    mlp = Mlp(gpu, m, 528, 640, m, prompt)
    try:
        mlp.feed(3)
        mlp.launch()
        mlp.check()
    finally:
        mlp.free()


@pytest.mark.parametrize("m,prompt", FORMS[1:])
def test_mlp_graph(gpu, m, prompt):
    """Replays on new inputs, with eager launches between, equal the eager
    results bit for bit."""
    mlp = Mlp(gpu, m, 528, 640, m, prompt)
    want = []
    for seed in range(4):
        mlp.feed(100 + 2 * seed)
        mlp.launch()
        want.append(mlp.results())
    graph = gpu.graph([hb.Op(k, ranges, m) for k, ranges, m in mlp.steps])
    try:
        for turn in range(3):
            for seed in (2, 0, 3, 1):
                mlp.feed(100 + 2 * seed)
                graph.launch()
                assert all(np.array_equal(a, b) for a, b in zip(mlp.results(), want[seed])), (turn, seed)
            mlp.feed(100)
            mlp.launch()
            gpu.sync()
    finally:
        graph.free()
        mlp.free()


def test_two_contexts(gpu):
    """Two contexts' launches in flight at once give each its own results, the
    split product's workspaces too."""
    other = hb.Gpu(0)
    mlps = []
    try:
        for g, seed in ((gpu, 5), (other, 6)):
            mlps += [Mlp(g, 40, 528, 640, seed, True), Mlp(g, 3, 528, 640, seed, False)]
        for i, mlp in enumerate(mlps):
            mlp.feed(50 + i)
            mlp.launch()
            mlp.check()
        alone = []
        for i, mlp in enumerate(mlps):
            mlp.feed(50 + i)
            mlp.launch()
            alone.append(mlp.results())
        for i, mlp in enumerate(mlps):
            mlp.feed(50 + i)
        for mlp in mlps:
            mlp.launch()
        for mlp, want in zip(mlps, alone):
            assert all(np.array_equal(a, b) for a, b in zip(mlp.results(), want))
    finally:
        for mlp in mlps[:2]:
            mlp.free()
        other.close()


# ---- the MoE layer and block ----

def check_experts(gpu, layer, m, gu, dn):
    """layer.buf's x rows, h and y against 64 bits, the combine against the
    oracle, over the m rows that just ran."""
    b, k, h, mi = layer.buf, layer.k, layer.h, layer.mi
    pairs, mv = m * k, layer.bm == 16
    sums = f8.sum_bound if mv else f8.mfma_bound
    route = gpu.download(b["route"], np.uint32, m * 2 * k).reshape(m, 2 * k)
    lst = gpu.download(b["list"], np.uint32, pairs)
    x = gpu.download(b["x"], np.uint16, m * h).reshape(m, h)
    hrow = 2 * mi if mv else hb.f8_row_bytes(mi)
    hraw = gpu.download(b["ehb"], np.uint8, pairs * hrow).reshape(pairs, hrow)
    ey = gpu.download(b["ey"], np.uint16, pairs * h).reshape(pairs, h)
    assert np.array_equal(np.sort(lst), np.arange(pairs))
    xv = f8.row_values(*f8.quantize_rows(x))
    if not mv:
        raw = gpu.download(b["xs"], np.uint8, m * hb.f8_row_bytes(h))
        assert np.array_equal(f8.row_values(*f8.unpack_rows(raw, m, h)), xv)
    e = route[:, :k].reshape(-1)[lst]
    for ex in np.unique(e):
        p = np.flatnonzero(e == ex)
        want, bound = swiglu_of(xv[lst[p] // k], gu[ex], sums)
        if mv:
            bits = np.ascontiguousarray(hraw[p]).view(np.uint16)
            f8.close(bits, want, bound, "h of expert %d" % ex)
            hv = f8.row_values(*f8.quantize_rows(bits))
        else:
            check_h(hraw[p], len(p), mi, want, bound)
            hv = f8.row_values(*f8.unpack_rows(hraw[p], len(p), mi))
        wv = f8.values(*dn[ex])
        f8.close(ey[lst[p]], hv @ wv.T, sums(hv, wv), "y of expert %d" % ex)
    out = gpu.download(b["out"], np.uint16, m * h).reshape(m, h)
    assert np.array_equal(out, orc.combine(ey, route, k, h))
    return out


def experts_of(rng, E, H, MI):
    return [f8.random_weights(rng, 2 * MI, H) for _ in range(E)], [f8.random_weights(rng, H, MI) for _ in range(E)]


@pytest.mark.parametrize("rows,bm", [(1, 16), (4, 16), (40, 32), (500, 64), (900, 128)])
def test_moe_layer(gpu, rows, bm):
    """The layer's ops, its two-call run over fewer rows, and the run that
    allocates nothing, which gives the same bits."""
    E, K, H, MI = 64, 4, 272, 128
    rng = np.random.default_rng(rows)
    gu, dn = experts_of(rng, E, H, MI)
    wg, wd, out = packed(gpu, gu), packed(gpu, dn), gpu.alloc(rows * H * 2)
    with hb.Engine(gpu, "") as e:
        layer = hb.MoeLayer(gpu, e, E, K, H, MI, rows, wg, wd, scores=hb.normal_bf16(1, 1.0, (rows, E)), x=hb.normal_bf16(2, 1.0, (rows, H)), f8=True)
        assert "experts" not in e.log() and layer.bm == bm
    try:
        gpu.time_ops(layer.ops(), 1)
        want = check_experts(gpu, layer, rows, gu, dn)
        gpu.zero(layer.buf["out"])
        layer.run()
        gpu.sync()
        assert np.array_equal(gpu.download(layer.buf["out"], np.uint16, rows * H).reshape(rows, H), want)
        m = max(1, rows // 2 - 3)
        gpu.upload(layer.buf["state"], np.array([0, 0, 0, m], np.uint32))
        layer.run(m)
        gpu.sync()
        want = check_experts(gpu, layer, m, gu, dn)
        hb.check(run_static(gpu, layer, out, m))
        gpu.sync()
        assert np.array_equal(gpu.download(out, np.uint16, m * H).reshape(m, H), want)
    finally:
        layer.free()
        for b in (wg, wd, out):
            gpu.free(b)


@pytest.mark.parametrize("rows,f8_experts", [(2, True), (60, True), (33, False)])
def test_moe_layer_routed(gpu, rows, f8_experts):
    """Sigmoid scores in f32 with biases and groups of experts, some of a row's
    masked: the route by its definition, and the layer behind it."""
    E, K, H, MI = 64, 6, 256, 128
    rng = np.random.default_rng(rows)
    s, bias = rng.normal(0, 1.5, (rows, E)).astype(np.float32), rng.normal(0, 0.1, E).astype(np.float32)
    s[0, 9:] = -np.inf
    kw = dict(score=hb.Score.Sigmoid, groups=8, top_groups=3, group_top=2, renorm=True, scale=2.5)
    bb = gpu.alloc_with(bias)
    gu, dn = experts_of(rng, E, H, MI)
    if f8_experts:
        wg, wd = packed(gpu, gu), packed(gpu, dn)
    else:
        wg, wd = gpu.alloc_with(hb.normal_bf16(1, 0.02, (E * 2 * MI, H))), gpu.alloc_with(hb.normal_bf16(2, 0.02, (E * H, MI)))
    x = hb.normal_bf16(2, 1.0, (rows, H))
    with hb.Engine(gpu, "") as e:
        layer = hb.MoeLayer(gpu, e, E, K, H, MI, rows, wg, wd, scores=s, x=x, f8=f8_experts,
                            route=hb.route_topk(E, K, bias=True, f32=True, **kw), bias=bb)
    try:
        gpu.zero(layer.buf["route"])
        layer.run()
        gpu.sync()
        got = gpu.download(layer.buf["route"], np.uint32, rows * 2 * K).reshape(rows, 2 * K)
        ids, w = route_ref(s, bias, top_k=K, **kw)
        assert np.array_equal(got[:, :K], ids)
        off = np.abs(np.ascontiguousarray(got[:, K:]).view(np.float32) - w)
        assert (off <= 48 * 2.0 ** -24 * np.abs(w) + 2.0 ** -140).all()
        if f8_experts:
            check_experts(gpu, layer, rows, gu, dn)
        else:
            ey = gpu.download(layer.buf["ey"], np.uint16, rows * K * H).reshape(rows * K, H)
            assert np.array_equal(gpu.download(layer.buf["out"], np.uint16, rows * H).reshape(rows, H), orc.combine(ey, got, K, H))
    finally:
        layer.free()
        for b in (wg, wd, bb):
            gpu.free(b)


@pytest.mark.parametrize("rows,biased", [(4, False), (24, True)])
def test_moe_block_from_checkpoint(gpu, tmp_path, rows, biased):
    """A checkpoint's experts quantised as they are uploaded, in the block that
    the bf16 path runs too."""
    from st_writer import write_model
    L, E, K, H, MI, SI = 1, 64, 4, 256, 128, 128
    p = "model.language_model.layers.%d." % L
    host = {"gu": hb.normal_bf16(93, 0.02, (E, 2 * MI, H)), "dn": hb.normal_bf16(94, 0.02, (E, H, MI))}
    write_model(str(tmp_path / "m"), [
        {p + "post_attention_layernorm.weight": ("BF16", hb.normal_bf16(91, 0.1, (H,))),
         p + "mlp.gate.weight": ("BF16", hb.normal_bf16(92, 0.05, (E, H))),
         p + "mlp.experts.gate_up_proj": ("BF16", host["gu"]),
         p + "mlp.experts.down_proj": ("BF16", host["dn"]),
         p + "mlp.shared_expert.gate_proj.weight": ("BF16", hb.normal_bf16(95, 0.02, (SI, H))),
         p + "mlp.shared_expert.up_proj.weight": ("BF16", hb.normal_bf16(96, 0.02, (SI, H))),
         p + "mlp.shared_expert.down_proj.weight": ("BF16", hb.normal_bf16(97, 0.02, (H, SI))),
         p + "mlp.shared_expert_gate.weight": ("BF16", hb.normal_bf16(98, 0.05, (1, H)))}])
    x0 = hb.normal_bf16(99, 1.0, (rows, H))
    route = hb.route_topk(E, K, score=hb.Score.Sigmoid, bias=True, f32=True) if biased else None
    with hb.Checkpoint(str(tmp_path / "m")) as ck, hb.Engine(gpu, "") as e:
        with pytest.raises(hb.HerbertError, match="upload_f8"):
            ck.upload_f8(gpu, [("%d.mlp.experts.down_proj" % L, E * H * MI)], MI, H, E - 1)
        w = hb.moe_weights_from_checkpoint(gpu, ck, L, E, H, MI, SI, f8=True)
        if biased:
            w["route_bias"] = gpu.alloc_with(np.linspace(-0.3, 0.3, E).astype(np.float32))
        block = hb.MoeBlock(gpu, e, E, K, H, MI, SI, rows, w, x0, f8=True, route=route)
    try:
        gpu.upload(block.buf["x"], x0)
        gpu.time_ops(block.ops(), 1)
        check_experts(gpu, block.layer, rows, [f8.quantize(t) for t in host["gu"]], [f8.quantize(t) for t in host["dn"]])
        assert not np.array_equal(gpu.download(block.buf["x"], np.uint16, rows * H).reshape(rows, H), x0)
    finally:
        block.free()
        for b in w.values():
            gpu.free(b)


def test_moe_layer_refuses(gpu):
    """A route of other experts, a bias without its route, both kinds of weights
    at once, and kernels that do not belong together."""
    E, K, H, MI, rows = 64, 4, 256, 128, 40
    wg, wd = gpu.alloc(E * hb.f8_bytes(H, 2 * MI)), gpu.alloc(E * hb.f8_bytes(MI, H))
    with hb.Engine(gpu, "") as e:
        for kw in (dict(route=hb.route_topk(E, K + 1)), dict(route=hb.route_topk(E // 2, K)), dict(bias=wg), dict(q4_group=32),
                   dict(route=hb.route_topk(E, K, bias=True))):
            with pytest.raises(hb.HerbertError, match="MoeLayer"):
                hb.MoeLayer(gpu, e, E, K, H, MI, rows, wg, wd, f8=True, **kw)
        layer = hb.MoeLayer(gpu, e, E, K, H, MI, rows, wg, wd, f8=True)
    sort, gu, dn, quantize = layer.kernels
    sort16 = gpu.pipeline(hb.Desc(kind=hb.Kind.SORT, experts=E, top_k=K, bm=16, rows_max=rows))
    gu16 = gpu.pipeline(hb.experts_f8(H, 2 * MI, hb.Out.Swiglu, hb.Rows.Gather, K, E, rows, 16))
    sums = gpu.pipeline(hb.experts_f8(H, 2 * MI, hb.Out.Bf16, hb.Rows.Gather, K, E, rows, 32))
    other = gpu.pipeline(hb.f8_quantize_rows(2 * H))
    gather = gpu.pipeline(hb.Desc(kind=hb.Kind.GATHER, n=H, top_k=K))
    try:
        for ks in ([sort16, gu, dn, quantize], [sort, gu16, dn, quantize], [sort, gu, gu, quantize], [sort, gu, dn, -1], [sort, gu, dn, other],
                   [sort, gu, dn, gather], [sort, sums, dn, quantize]):
            rc = hb.lib.hb_moe_experts_run(gpu.h, (ctypes.c_int32 * 4)(*ks), layer.swiglu_k, layer.combine_k, ctypes.byref(layer.io),
                                           hb.r(layer.buf["out"]), rows)
            assert rc == hb.ERR_INVALID and "moe experts" in hb.last_error(), ks
    finally:
        layer.free()
        gpu.free(wg)
        gpu.free(wd)


# ---- a prompt's MLP ----

def test_prefill_mlp_from_checkpoint(gpu, tmp_path):
    """A prompt in blocks over a checkpoint's weights in 8 bits: the last block's
    steps each on the input it had, and the first block as it is alone."""
    from st_writer import write_model
    h, inter, n = 512, 768, 300
    gate, up = hb.normal_bf16(71, 0.02, (inter, h)), hb.normal_bf16(72, 0.02, (inter, h))
    down, pn = hb.normal_bf16(73, 0.02, (h, inter)), hb.normal_bf16(74, 0.1, (h,))
    p = "model.language_model.layers.3."
    write_model(str(tmp_path / "m"), [{p + "mlp.gate_proj.weight": ("BF16", gate), p + "post_attention_layernorm.weight": ("BF16", pn),
                                       p + "mlp.up_proj.weight": ("BF16", up), p + "mlp.down_proj.weight": ("BF16", down)}])
    x0 = hb.normal_bf16(75, 1.0, (n, h))
    with hb.Checkpoint(str(tmp_path / "m")) as ck, hb.Engine(gpu, "prefill.block=128") as e:
        mlp = hb.PrefillMlp(gpu, e, ck, 3, h, inter, f8=True)
    X = gpu.alloc_with(x0)
    states, first = mlp.states(n), mlp.states(128)
    try:
        gpu.time_ops(mlp.ops(X, n, states), 1)
        got = gpu.download(X, np.uint16, n * h).reshape(n, h)
        m = n - 256
        xn = gpu.download(mlp.buf["xn"], np.uint16, m * h).reshape(m, h)
        t = f8.f64(x0[256:])
        t = t / np.sqrt((t * t).mean(-1, keepdims=True) + 1e-6) * (f8.f64(pn) + 1)
        f8.close(xn, t, 32 * f8.U * np.abs(t), "norm")  # its roundings, at most 32 reach a value
        raw = gpu.download(mlp.buf["x8"], np.uint8, m * hb.f8_row_bytes(h))
        xv = f8.row_values(*f8.quantize_rows(xn))
        assert np.array_equal(f8.row_values(*f8.unpack_rows(raw, m, h)), xv)
        raw = gpu.download(mlp.buf["h8"], np.uint8, m * hb.f8_row_bytes(inter))
        check_h(raw.reshape(m, -1), m, inter, *swiglu_of(xv, f8.quantize(np.concatenate([gate, up])), f8.mfma_bound))
        hv, wv = f8.row_values(*f8.unpack_rows(raw, m, inter)), f8.values(*f8.quantize(down))
        want = hv @ wv.T + f8.f64(x0[256:])
        f8.close(got[256:], want, f8.mfma_bound(hv, wv) + f8.U * np.abs(want), "down")
        gpu.upload(X, x0)
        gpu.time_ops(mlp.ops(X, 128, first), 1)
        assert np.array_equal(gpu.download(X, np.uint16, 128 * h).reshape(128, h), got[:128])
    finally:
        for b in states + first + [X]:
            gpu.free(b)
        mlp.free()


# ---- large sizes ----

def test_matrix_past_4_gib(gpu):
    """Codes past 2^32 bytes: rows on both sides of it and the last one."""
    k, n = 16384, 262789
    assert hb.f8_bytes(k, n) > 1 << 32
    rng = np.random.default_rng(4)
    at = [0, 17, 131071, 131072, 262143, 262144, n - 1]  # 2^31 and 2^32 code bytes are 131072 and 262144 rows
    w, q = gpu.alloc(n * k * 2), gpu.alloc(hb.f8_bytes(k, n))
    x = f8.exact_x(rng, 1, k, (0, 1))
    y, xb = gpu.alloc(n * 4), gpu.alloc_with(x)
    try:
        gpu.zero(w)
        # Wholes of -2..2 and a 448 in each block of a row: scales of 1, sums that
        # f32 holds.
        rows = rng.integers(-2, 3, (len(at), k)).astype(np.float32)
        rows[:, ::128] = 448
        for r, row in zip(at, rows):
            gpu.upload(w, hb.f32_to_bf16(row), r * k * 2)
        gpu.launch(gpu.pipeline(hb.f8_quantize(k, n)), [hb.r(w), hb.r(q)], 1)
        gpu.launch(gpu.pipeline(hb.matvec_f8(k, n, hb.Out.F32)), [hb.r(q), hb.r(xb), hb.r(y)], 1)
        got = gpu.download(y, np.float32, n)
        want = np.zeros(n)
        want[at] = rows.astype(np.float64) @ f8.f64(x[0])
        assert (np.abs(rows).astype(np.float64) @ np.abs(f8.f64(x[0]))).max() < 2 ** 24
        assert np.array_equal(got, want)
        gpu.upload(w, np.full(k, 0x4242, np.uint16), at[-1] * k * 2)
        gpu.launch(gpu.pipeline(hb.f8_dequantize(k, n)), [hb.r(q), hb.r(w)], 1)
        for r, row in zip(at, rows):
            assert np.array_equal(hb.bf16_to_f32(gpu.download(w, np.uint16, k, r * k * 2)), row), r
    finally:
        for b in (w, q, y, xb):
            gpu.free(b)


def test_native_host(gpu):
    r = subprocess.run([os.path.join(ROOT, "herbert-metal-bf16_amd", "hb_gemm"), "--reps", "3", "f8:3x1024x256f", "f8:50x528x64"],
                       capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stderr
    lines = r.stdout.splitlines()
    assert lines[0].startswith("f8:3x1024x256 matvec_f8_1024x256_f32_") and lines[1].startswith("f8:50x528x64 gemm_f8_528x64_")
