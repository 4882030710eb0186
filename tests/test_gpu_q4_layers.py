"""The 4-bit operators as they are used together: a decode layer from norm to
norm (eager, and recorded into a graph beside eager work), the MoE layer and
block over packed experts, two contexts at once, a matrix past 4 GiB, and the
native host."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import herbert_hip as hb
import hb_oracle as orc
import q4_ref as q4
from test_zz_no_alloc import run_static

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EPS = 1e-6


def f64(bits):
    return hb.bf16_to_f32(bits).astype(np.float64)


def rms(t, w):
    return t / np.sqrt((t * t).mean(-1, keepdims=True) + EPS) * (f64(w) + 1)


class Layer:
    """A decode layer over packed weights: norm, qkv, o of the q part (the
    attention between them is the caller's), post norm and residual add and
    next norm, gate|up with the SwiGLU, down, residual add and next norm."""

    def __init__(self, gpu, engine, m, h, q, kv, inter, group, seed):
        self.gpu, self.m, self.h, self.q, self.inter, self.group = gpu, m, h, q, inter, group
        rng = np.random.default_rng(seed)
        self.host, self.b = {}, {}
        for name, n, k in (("qkv", q + 2 * kv, h), ("o", h, q), ("gate_up", 2 * inter, h), ("down", h, inter)):
            codes, scales = q4.random_codes(rng, n, k, group)
            self.host[name] = (codes, scales)
            self.b[name] = q4.pack(gpu, codes, scales, k, n, group)
        for name in ("n0", "n1", "n2", "n3"):
            self.host[name] = hb.normal_bf16(seed + len(self.host), 0.1, h)
            self.b[name] = gpu.alloc_with(self.host[name])
        for name, width in (("x", h), ("xn", h), ("qkv_y", q + 2 * kv), ("ao", q), ("oy", h), ("x1", h), ("h1", h),
                            ("hh", inter), ("dy", h), ("x2", h), ("h2", h)):
            self.b[name] = gpu.alloc(m * width * 2)
        b = {name: hb.r(v) for name, v in self.b.items()}
        mv = lambda w, n, k, out, x, y: (engine.mv_q4(k, n, out, group, m, [b[w]], b[x], b[y]), [b[w], b[x], b[y]], m)  # noqa: E731
        norm = gpu.pipeline(hb.block_norm(h, EPS, True, post=True, pre=True))
        add = gpu.pipeline(hb.block_norm(h, EPS, True))
        self.steps = [(gpu.pipeline(hb.rmsnorm(h, EPS, True)), [b["x"], b["n0"], b["xn"]], m),
                      mv("qkv", q + 2 * kv, h, hb.Out.Bf16, "xn", "qkv_y"),
                      mv("o", h, q, hb.Out.Bf16, "ao", "oy"),
                      (norm, [b["x"], b["oy"], b["x1"], b["h1"], b["n1"], b["n2"]], m),
                      mv("gate_up", 2 * inter, h, hb.Out.Swiglu, "h1", "hh"),
                      mv("down", h, inter, hb.Out.Bf16, "hh", "dy"),
                      (add, [b["x1"], b["dy"], b["x2"], b["h2"], b["n3"]], m)]

    def feed(self, seed):
        self.gpu.upload(self.b["x"], hb.normal_bf16(seed, 1.0, (self.m, self.h)))
        self.gpu.upload(self.b["ao"], hb.normal_bf16(seed + 1, 1.0, (self.m, self.q)))

    def launch(self):
        for k, ranges, m in self.steps:
            self.gpu.launch(k, ranges, m)

    def get(self, name):
        return self.gpu.download(self.b[name], np.uint16, self.gpu.size(self.b[name]) // 2).reshape(self.m, -1)

    def results(self):
        self.gpu.sync()
        return {n: self.get(n) for n in ("qkv_y", "x1", "hh", "x2", "h2")}

    def check(self):
        """Every step against 64 bits on the input it had."""
        v = {n: self.get(n) for n in ("x", "xn", "qkv_y", "ao", "oy", "x1", "h1", "hh", "dy", "x2", "h2")}

        def lin(w, x):
            c, s = self.host[w]
            return f64(x) @ q4.values(c, s, self.group).T, q4.sum_bound(f64(x), c, s, self.group)

        q4.close(v["qkv_y"], *lin("qkv", v["xn"]), "qkv")
        q4.close(v["oy"], *lin("o", v["ao"]), "o")
        # f32 arithmetic of the norms: 32 roundings at most reach a value.
        t = rms(f64(v["oy"]), self.host["n1"])
        q4.close(v["x1"], f64(v["x"]) + t, 32 * q4.U * (np.abs(f64(v["x"])) + np.abs(t)), "x1")
        t = rms(f64(v["x1"]), self.host["n2"])
        q4.close(v["h1"], t, 32 * q4.U * np.abs(t), "h1")
        both, e = lin("gate_up", v["h1"])
        g, u, n = both[:, :self.inter], both[:, self.inter:], self.inter
        q4.close(v["hh"], q4.silu(g) * u, q4.swiglu_bound(g, u, e[:, :n], e[:, n:]), "h")
        q4.close(v["dy"], *lin("down", v["hh"]), "down")
        q4.close(v["x2"], f64(v["x1"]) + f64(v["dy"]), q4.U * np.abs(f64(v["x1"]) + f64(v["dy"])), "x2")
        t = rms(f64(v["x2"]), self.host["n3"])
        q4.close(v["h2"], t, 32 * q4.U * np.abs(t), "h2")

    def free(self):
        for buf in self.b.values():
            self.gpu.free(buf)


@pytest.mark.parametrize("m,group", [(1, 32), (4, 64), (9, 128)])
def test_decode_layer(gpu, m, group):
    with hb.Engine(gpu, "") as e:
        layer = Layer(gpu, e, m, 512, 768, 128, 640, group, 40 + m)
    try:
        layer.feed(7)
        layer.launch()
        gpu.sync()
        layer.check()
    finally:
        layer.free()


def test_decode_layer_graph(gpu):
    """Replays on new inputs, with eager launches between, equal the eager
    results bit for bit."""
    with hb.Engine(gpu, "mv.auto=0") as e:
        layer = Layer(gpu, e, 2, 512, 768, 128, 640, 32, 3)
    want = []
    for seed in range(4):
        layer.feed(100 + seed)
        layer.launch()
        want.append(layer.results())
    graph = gpu.graph([hb.Op(k, ranges, m) for k, ranges, m in layer.steps])
    try:
        for turn in range(3):
            for seed in (2, 0, 3, 1):
                layer.feed(100 + seed)
                graph.launch()
                got = layer.results()
                assert all(np.array_equal(got[n], want[seed][n]) for n in got), (turn, seed)
            layer.feed(100)
            layer.launch()
            gpu.sync()
    finally:
        graph.free()
        layer.free()


def test_two_contexts(gpu):
    """Two contexts' launches in flight at once give each its own results."""
    other = hb.Gpu(0)
    layers = []
    try:
        for g, seed in ((gpu, 5), (other, 6)):
            with hb.Engine(g, "mv.auto=0") as e:
                layers.append(Layer(g, e, 3, 512, 768, 128, 640, 64, seed))
        alone = []
        for i, layer in enumerate(layers):
            layer.feed(50 + i)
            layer.launch()
            alone.append(layer.results())
        for _ in range(20):
            for layer in layers:
                layer.launch()
        for layer, want in zip(layers, alone):
            got = layer.results()
            assert all(np.array_equal(got[n], want[n]) for n in got)
    finally:
        if layers:
            layers[0].free()
        other.close()


# ---- the MoE layer and block ----

def check_experts(gpu, layer, m, gu, gs, dn, ds, group):
    """layer.buf's h and y rows against 64 bits, the combine against the
    oracle, over the m rows that just ran."""
    b, k, h, mi = layer.buf, layer.k, layer.h, layer.mi
    pairs = m * k
    route = gpu.download(b["route"], np.uint32, m * 2 * k).reshape(m, 2 * k)
    lst = gpu.download(b["list"], np.uint32, pairs)
    x = gpu.download(b["x"], np.uint16, m * h).reshape(m, h)
    hh = gpu.download(b["ehb"], np.uint16, pairs * mi).reshape(pairs, mi)
    ey = gpu.download(b["ey"], np.uint16, pairs * h).reshape(pairs, h)
    assert np.array_equal(np.sort(lst), np.arange(pairs))
    e = route[:, :k].reshape(-1)[lst]
    for ex in np.unique(e):
        p = np.flatnonzero(e == ex)
        c, s = gu[ex * 2 * mi:(ex + 1) * 2 * mi], gs[ex * 2 * mi:(ex + 1) * 2 * mi]
        xf = f64(x[lst[p] // k])
        both, eb = xf @ q4.values(c, s, group).T, q4.sum_bound(xf, c, s, group)
        g, u = both[:, :mi], both[:, mi:]
        q4.close(hh[p], q4.silu(g) * u, q4.swiglu_bound(g, u, eb[:, :mi], eb[:, mi:]), "h of expert %d" % ex)
        c, s = dn[ex * h:(ex + 1) * h], ds[ex * h:(ex + 1) * h]
        hf = f64(hh[p])
        q4.close(ey[lst[p]], hf @ q4.values(c, s, group).T, q4.sum_bound(hf, c, s, group), "y of expert %d" % ex)
    out = gpu.download(b["out"], np.uint16, m * h).reshape(m, h)
    assert np.array_equal(out, orc.combine(ey, route, k, h))
    return out


@pytest.mark.parametrize("rows,group", [(1, 32), (40, 64), (200, 128)])
def test_moe_layer(gpu, rows, group):
    """The layer's ops, its two-call run over fewer rows, and the run that
    allocates nothing, which gives the same bits."""
    E, K, H, MI = 64, 4, 256, 128
    rng = np.random.default_rng(rows)
    gu, gs = q4.random_codes(rng, E * 2 * MI, H, group)
    dn, ds = q4.random_codes(rng, E * H, MI, group)
    wg, wd = q4.pack(gpu, gu, gs, H, 2 * MI, group, E), q4.pack(gpu, dn, ds, MI, H, group, E)
    out = gpu.alloc(rows * H * 2)
    with hb.Engine(gpu, "") as e:
        layer = hb.MoeLayer(gpu, e, E, K, H, MI, rows, wg, wd, scores=hb.normal_bf16(1, 1.0, (rows, E)),
                            x=hb.normal_bf16(2, 1.0, (rows, H)), q4_group=group)
        assert "experts" not in e.log()
    try:
        gpu.time_ops(layer.ops(), 1)
        want = check_experts(gpu, layer, rows, gu, gs, dn, ds, group)
        gpu.zero(layer.buf["out"])
        layer.run()
        gpu.sync()
        assert np.array_equal(gpu.download(layer.buf["out"], np.uint16, rows * H).reshape(rows, H), want)
        m = max(1, rows // 2 - 3)
        gpu.upload(layer.buf["state"], np.array([0, 0, 0, m], np.uint32))
        layer.run(m)
        gpu.sync()
        want = check_experts(gpu, layer, m, gu, gs, dn, ds, group)
        hb.check(run_static(gpu, layer, out, m))
        gpu.sync()
        assert np.array_equal(gpu.download(out, np.uint16, m * H).reshape(m, H), want)
    finally:
        layer.free()
        for b in (wg, wd, out):
            gpu.free(b)


def test_moe_run_with_the_swiglu_apart(gpu):
    """A gate|up that writes its sums (Out::Bf16), then swiglu_slots: h from
    the rounded sums, everything else as in the fused run."""
    E, K, H, MI, rows, group = 64, 4, 256, 128, 21, 64
    rng = np.random.default_rng(12)
    gu, gs = q4.random_codes(rng, E * 2 * MI, H, group)
    dn, ds = q4.random_codes(rng, E * H, MI, group)
    wg, wd = q4.pack(gpu, gu, gs, H, 2 * MI, group, E), q4.pack(gpu, dn, ds, MI, H, group, E)
    with hb.Engine(gpu, "") as e:
        layer = hb.MoeLayer(gpu, e, E, K, H, MI, rows, wg, wd, scores=hb.normal_bf16(1, 1.0, (rows, E)),
                            x=hb.normal_bf16(2, 1.0, (rows, H)), q4_group=group)
    b, pairs = layer.buf, rows * K
    try:
        layer.kernels[1] = gpu.pipeline(hb.experts_q4(H, 2 * MI, hb.Out.Bf16, group, hb.Rows.Gather, K, E, rows))
        layer.run()
        gpu.sync()
        egu = gpu.download(b["egu"], np.uint16, pairs * 2 * MI).reshape(pairs, 2 * MI)
        hh = gpu.download(b["ehb"], np.uint16, pairs * MI).reshape(pairs, MI)
        assert np.array_equal(hh, orc.swiglu(egu, MI))
        route = gpu.download(b["route"], np.uint32, rows * 2 * K).reshape(rows, 2 * K)
        lst = gpu.download(b["list"], np.uint32, pairs)
        x, ey = gpu.download(b["x"], np.uint16, rows * H).reshape(rows, H), gpu.download(b["ey"], np.uint16, pairs * H).reshape(pairs, H)
        e = route[:, :K].reshape(-1)[lst]
        for ex in np.unique(e):
            p = np.flatnonzero(e == ex)
            for got, xf, c, s in ((egu[p], f64(x[lst[p] // K]), gu[ex * 2 * MI:][:2 * MI], gs[ex * 2 * MI:][:2 * MI]),
                                  (ey[lst[p]], f64(hh[p]), dn[ex * H:][:H], ds[ex * H:][:H])):
                q4.close(got, xf @ q4.values(c, s, group).T, q4.sum_bound(xf, c, s, group), "expert %d" % ex)
        assert np.array_equal(gpu.download(b["out"], np.uint16, rows * H).reshape(rows, H), orc.combine(ey, route, K, H))
    finally:
        layer.free()
        gpu.free(wg)
        gpu.free(wd)


def test_moe_run_refuses(gpu):
    """Kernels that do not belong together: a sort of other tiles, the gate|up
    and down rows swapped, one bf16 and one 4-bit kernel, a gather kernel."""
    E, K, H, MI, rows, group = 64, 4, 256, 128, 8, 32
    wg, wd = gpu.alloc(E * hb.q4_bytes(H, 2 * MI, group)), gpu.alloc(E * hb.q4_bytes(MI, H, group))
    with hb.Engine(gpu, "") as e:
        layer = hb.MoeLayer(gpu, e, E, K, H, MI, rows, wg, wd, q4_group=group)
    good = layer.kernels
    sort32 = gpu.pipeline(hb.Desc(kind=hb.Kind.SORT, experts=E, top_k=K, bm=32, rows_max=rows))
    swapped = gpu.pipeline(hb.experts_q4(H, 2 * MI, hb.Out.Swiglu, group, hb.Rows.Scatter, K, E, rows))
    bf16 = gpu.pipeline(hb.gemm_mma_rows(MI, H, hb.Out.Bf16, rows_of=hb.Rows.Scatter, top_k=K, experts=E, bm=16,
                                         tiles=hb.moe_tiles(rows, K, E, 16), wm=1, wn=4, bn=128, bk=64, rows_max=rows))
    gather = gpu.pipeline(hb.Desc(kind=hb.Kind.GATHER, n=H, top_k=K))
    try:
        for ks in ([sort32] + good[1:], [good[0], swapped] + good[2:], good[:2] + [bf16, -1], good[:3] + [gather],
                   [good[0], good[1], good[1], -1]):
            rc = hb.lib.hb_moe_experts_run(gpu.h, (ctypes.c_int32 * 4)(*ks), layer.swiglu_k, layer.combine_k,
                                           ctypes.byref(layer.io), hb.r(layer.buf["out"]), rows)
            assert rc == hb.ERR_INVALID and "moe experts" in hb.last_error(), ks
    finally:
        layer.free()
        gpu.free(wg)
        gpu.free(wd)


def test_moe_block_from_checkpoint(gpu, tmp_path):
    """A checkpoint's experts quantised as they are uploaded, in the block that
    the bf16 path runs too."""
    from st_writer import write_model
    L, E, K, H, MI, SI, rows, group = 1, 64, 4, 256, 128, 128, 24, 32
    p = "model.language_model.layers.%d." % L
    host = {"gu": hb.normal_bf16(93, 0.02, (E * 2 * MI, H)), "dn": hb.normal_bf16(94, 0.02, (E * H, MI))}
    write_model(str(tmp_path / "m"), [
        {p + "post_attention_layernorm.weight": ("BF16", hb.normal_bf16(91, 0.1, (H,))),
         p + "mlp.gate.weight": ("BF16", hb.normal_bf16(92, 0.05, (E, H))),
         p + "mlp.experts.gate_up_proj": ("BF16", host["gu"].reshape(E, 2 * MI, H)),
         p + "mlp.experts.down_proj": ("BF16", host["dn"].reshape(E, H, MI)),
         p + "mlp.shared_expert.gate_proj.weight": ("BF16", hb.normal_bf16(95, 0.02, (SI, H))),
         p + "mlp.shared_expert.up_proj.weight": ("BF16", hb.normal_bf16(96, 0.02, (SI, H))),
         p + "mlp.shared_expert.down_proj.weight": ("BF16", hb.normal_bf16(97, 0.02, (H, SI))),
         p + "mlp.shared_expert_gate.weight": ("BF16", hb.normal_bf16(98, 0.05, (1, H)))}])
    x0 = hb.normal_bf16(99, 1.0, (rows, H))
    with hb.Checkpoint(str(tmp_path / "m")) as ck, hb.Engine(gpu, "") as e:
        with pytest.raises(hb.HerbertError, match="upload_q4"):
            ck.upload_q4(gpu, [("%d.mlp.experts.down_proj" % L, E * H * MI)], MI, H, group, E - 1)
        w = hb.moe_weights_from_checkpoint(gpu, ck, L, E, H, MI, SI, q4_group=group)
        block = hb.MoeBlock(gpu, e, E, K, H, MI, SI, rows, w, x0, q4_group=group)
    try:
        (gu, gs), (dn, ds) = q4.quantize(host["gu"], group), q4.quantize(host["dn"], group)
        gpu.upload(block.buf["x"], x0)
        gpu.time_ops(block.ops(), 1)
        check_experts(gpu, block.layer, rows, gu, gs, dn, ds, group)
        assert not np.array_equal(gpu.download(block.buf["x"], np.uint16, rows * H).reshape(rows, H), x0)
    finally:
        block.free()
        for b in w.values():
            gpu.free(b)


def test_matrix_past_4_gib(gpu):
    """Codes past 2^32 bytes: rows on both sides of it and the last one."""
    k, n, group = 16384, 589829, 128
    assert hb.q4_bytes(k, n, group) > 1 << 32
    rng = np.random.default_rng(4)
    at = [0, 17, 524271, 524272, 524288, 524304, n - 1]  # 2^32 code bytes are 524288 rows
    w, q = gpu.alloc(n * k * 2), gpu.alloc(hb.q4_bytes(k, n, group))
    y, x = gpu.alloc(n * 4), hb.f32_to_bf16(rng.integers(-2, 3, (1, k)).astype(np.float32))
    xb = gpu.alloc_with(x)
    try:
        gpu.zero(w)
        # Wholes of -8..7 with a -8 in each group: scales of 1, exact sums.
        rows = rng.integers(-8, 8, (len(at), k)).astype(np.float32)
        rows[:, ::group] = -8
        for r, row in zip(at, rows):
            gpu.upload(w, hb.f32_to_bf16(row), r * k * 2)
        gpu.launch(gpu.pipeline(hb.q4_quantize(k, n, group)), [hb.r(w), hb.r(q)], 1)
        gpu.launch(gpu.pipeline(hb.matvec_q4(k, n, hb.Out.F32, group)), [hb.r(q), hb.r(xb), hb.r(y)], 1)
        got = gpu.download(y, np.float32, n)
        want = np.zeros(n)
        want[at] = rows.astype(np.float64) @ hb.bf16_to_f32(x[0]).astype(np.float64)
        assert np.array_equal(got, want)
        gpu.upload(w, np.full(k, 0x4242, np.uint16), at[-1] * k * 2)
        gpu.launch(gpu.pipeline(hb.q4_dequantize(k, n, group)), [hb.r(q), hb.r(w)], 1)
        for r, row in zip(at, rows):
            assert np.array_equal(hb.bf16_to_f32(gpu.download(w, np.uint16, k, r * k * 2)), row), r
    finally:
        for b in (w, q, y, xb):
            gpu.free(b)


def test_native_host(gpu):
    r = subprocess.run([os.path.join(ROOT, "herbert-metal-bf16_amd", "hb_gemm"), "--reps", "3", "q4:3x1024x256f", "q4:1x520x64"],
                       capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stderr
    lines = r.stdout.splitlines()
    assert lines[0].startswith("q4:3x1024x256 matvec_q4_1024x256_g32_f32_") and lines[1].startswith("q4:1x520x64 matvec_q4_520x64_g32_")
