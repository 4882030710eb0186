"""What the library refuses of the 4-bit weights' kernels and block_norm, on
the CPU over a HIP runtime on host memory, and the forms that compile."""
import ctypes

import numpy as np
import pytest

import herbert_hip
import host_gpu


@pytest.fixture(scope="module")
def hb(tmp_path_factory):
    mp = pytest.MonkeyPatch()
    mp.setenv("HB_CACHE_DIR", "")
    yield host_gpu.load(tmp_path_factory.mktemp("host"))
    mp.undo()


@pytest.fixture()
def gpu(hb):
    g = hb.Gpu(0)
    yield g
    g.close()


def test_q4_bytes(hb):
    assert hb.q4_bytes(128, 16, 32) == 1024 + 512
    assert hb.q4_bytes(136, 17, 64) == 4 * 1024 + 2 * 256
    assert hb.q4_bytes(2560, 151936, 128) == 20 * 9496 * (1024 + 32)
    for k, n, g in [(0, 1, 32), (8, 0, 32), (12, 1, 32), (8, 1, 16), (8, 1, 0), (8, 1, 256)]:
        with pytest.raises(hb.HerbertError):
            hb.q4_bytes(k, n, g)


@pytest.mark.parametrize("make,match", [
    (lambda hb: hb.matvec_q4(100, 16, hb.Out.Bf16), "K a multiple of 8"),
    (lambda hb: hb.matvec_q4(128, 16, hb.Out.Bf16, group=48), "groups of"),
    (lambda hb: hb.matvec_q4(128, 16, hb.Out.Bf16, mv_m=17), "m <= 16"),
    (lambda hb: hb.matvec_q4(128, 16, 4), "out"),
    (lambda hb: hb.matvec_q4(128, 48, hb.Out.Swiglu), "multiple of 16"),
    (lambda hb: hb.matvec_q4(128, 64, hb.Out.Swiglu, rows=16), "rows a wave"),
    (lambda hb: hb.matvec_q4(128, 64, hb.Out.Bf16, rows=48), "rows a wave"),
    (lambda hb: hb.matvec_q4(128, 64, hb.Out.Bf16, waves=3), "waves"),
    (lambda hb: hb.matvec_q4(128, 64, hb.Out.Bf16, split=8, waves=4), "split"),
    (lambda hb: hb.matvec_q4(128, 64, hb.Out.Bf16, unroll=5), "unroll"),
    (lambda hb: hb.experts_q4(128, 64, hb.Out.F32, 32, hb.Rows.Gather, 8, 64, 4), "bf16 out"),
    (lambda hb: hb.experts_q4(128, 64, hb.Out.Bf16, 32, hb.Rows.Sorted, 8, 64, 4), "rows_of"),
    (lambda hb: hb.experts_q4(128, 64, hb.Out.Bf16, 32, hb.Rows.Gather, 8, 64, 4).replace(tiles=0), "tiles"),
    (lambda hb: hb.experts_q4(128, 64, hb.Out.Bf16, 32, hb.Rows.Gather, 8, 2048, 4), "experts"),
    (lambda hb: hb.experts_q4(128, 64, hb.Out.Bf16, 32, hb.Rows.Gather, 8, 64, 1 << 26), "pairs"),
    (lambda hb: hb.matvec_q4((1 << 20) + 8, 16, hb.Out.Bf16), "K a multiple of 8 up to"),
    (lambda hb: hb.matvec_q4(128, (1 << 24) + 1, hb.Out.Bf16), "N up to"),
    (lambda hb: hb.matvec_q4(1 << 20, 1 << 24, hb.Out.Bf16), "K N below"),
    (lambda hb: hb.q4_quantize(1 << 20, 1 << 24), "K N below"),
    (lambda hb: hb.q4_quantize(4, 16), "K a multiple of 8"),
    (lambda hb: hb.q4_pack(8, 16, 31), "groups"),
    (lambda hb: hb.q4_dequantize(8, 0), "q4"),
    (lambda hb: hb.block_norm(0, 1e-6), "rows of 1"),
    (lambda hb: hb.block_norm(32769, 1e-6), "rows of 1"),
    (lambda hb: hb.block_norm(64, 1e-6).replace(form=64), "parts"),
    (lambda hb: hb.block_norm(64, 1e-6).replace(form=8), "parts"),
])
def test_refused_descriptors(hb, gpu, make, match):
    with pytest.raises(hb.HerbertError, match=match):
        gpu.pipeline(make(hb))


def matvec_bufs(hb, gpu, k=128, n=32, m=2):
    return gpu.alloc(hb.q4_bytes(k, n)), gpu.alloc(m * k * 2 + 64), gpu.alloc(m * n * 4 + 64)


def test_refused_matvec_launches(hb, gpu):
    w, x, y = matvec_bufs(hb, gpu)
    k = gpu.pipeline(hb.matvec_q4(128, 32, hb.Out.F32, mv_m=2))
    R = hb.r
    gpu.launch(k, [R(w), R(x), R(y)], 2)
    gpu.launch(k, [R(w), R(x, 2), R(y, 4)], 2)
    for ranges, m, match in [([R(w), R(x), R(y)], 0, "0 rows"), ([R(w), R(x), R(y)], 3, "rows: 1..2"),
                             ([R(w, 0, 2559), R(x), R(y)], 1, "q4"), ([R(w), R(x, 0, 511), R(y)], 2, "binding 1"),
                             ([R(w), R(x), R(y, 0, 255)], 2, "binding 2"), ([R(w), R(x, 1), R(y)], 1, "multiple of 2"),
                             ([R(w), R(x), R(y, 2)], 1, "multiple of 4"), ([R(y), R(x), R(w, 8)], 1, "binding"),
                             ([R(w), R(x), R(x, 4)], 1, "overlap"), ([R(w), R(x), R(w, 1024)], 1, "overlap"),
                             ([R(w), R(x)], 1, "bindings given")]:
        with pytest.raises(hb.HerbertError, match=match):
            gpu.launch(k, ranges, m)
        if len(ranges) == 3:
            with pytest.raises(hb.HerbertError, match=match):
                gpu.graph([hb.Op(k, ranges, m)])
            with pytest.raises(hb.HerbertError, match=match):
                gpu.time_ops([hb.Op(k, ranges, m)])
    big = gpu.alloc(hb.q4_bytes(128, 32) + 32)
    with pytest.raises(hb.HerbertError, match="multiple of 16"):
        gpu.launch(k, [R(big, 8), R(x), R(y)], 1)


def test_refused_experts_launches(hb, gpu):
    t, top_k, experts = 4, 2, 16
    k = gpu.pipeline(hb.experts_q4(128, 64, hb.Out.Swiglu, 32, hb.Rows.Gather, top_k, experts, t))
    assert gpu.groups(k, 1) <= 2 * 2 and gpu.groups(k, t) <= 8 * 2
    sizes = [16, experts * hb.q4_bytes(128, 64), t * 128 * 2, t * top_k * 32 * 2, t * top_k * 4,
             (1 + 3 * hb.moe_tiles(t, top_k, experts, 16)) * 4]
    b = [gpu.alloc(s) for s in sizes]
    for i, s in enumerate(sizes):
        ranges = [hb.r(x) for x in b]
        ranges[i] = hb.r(b[i], 0, s - 1)
        with pytest.raises(hb.HerbertError, match="binding %d" % i):
            gpu.launch(k, ranges, t)
    with pytest.raises(hb.HerbertError, match="rows_max"):
        gpu.launch(k, [hb.r(x) for x in b], t + 1)


def test_refused_norm_launches(hb, gpu):
    n, m = 40, 3
    k = gpu.pipeline(hb.block_norm(n, 1e-6, post=True, gate=hb.Gate.Elements, scales=True))
    row = m * n * 2
    x, y, xo, h, g = (gpu.alloc(row + 64) for _ in range(5))
    wp, wn, sc = gpu.alloc(n * 2), gpu.alloc(n * 2), gpu.alloc(8)
    R = hb.r
    good = [R(x), R(y), R(xo), R(h), R(wp), R(g), R(sc), R(wn)]
    gpu.launch(k, good, m)
    for over in [{2: R(x)}, {2: R(y)}, {2: R(x), 3: R(y)}, {3: R(g)}, {3: R(x), 2: R(g)}]:
        gpu.launch(k, [over.get(i, v) for i, v in enumerate(good)], m)
    for bad, match in [({2: R(x, 2)}, "overlap"), ({3: R(xo)}, "overlap"), ({3: R(y, 16)}, "overlap"), ({2: R(g, 4)}, "overlap"),
                       ({0: R(x, 1)}, "multiple of 2"), ({6: R(sc, 0, 4)}, "scales"), ({4: R(wp, 0, 78)}, "w_post"),
                       ({7: R(wn, 0, 78)}, "w_pre"), ({5: R(g, 0, row - 2)}, "gate"), ({3: R(h, 0, row - 2)}, "binding 3")]:
        with pytest.raises(hb.HerbertError, match=match):
            gpu.launch(k, [bad.get(i, v) for i, v in enumerate(good)], m)
    with pytest.raises(hb.HerbertError, match="0 rows"):
        gpu.launch(k, good, 0)
    with pytest.raises(hb.HerbertError, match="too many rows"):
        gpu.launch(k, good, 1 << 26)
    many = gpu.pipeline(hb.experts_q4(8, 1 << 24, hb.Out.Bf16, 32, hb.Rows.Gather, 8, 64, 1 << 20))
    with pytest.raises(hb.HerbertError, match="too many workgroups"):
        gpu.launch(many, [R(x)] * 6, 1 << 20)


def test_refused_quantize_launches(hb, gpu):
    k = gpu.pipeline(hb.q4_quantize(64, 16))
    w, q = gpu.alloc(2 * 64 * 16), gpu.alloc(hb.q4_bytes(64, 16))
    for ranges, m, match in [([hb.r(w, 0, 2046), hb.r(q)], 1, "W"), ([hb.r(w), hb.r(q, 0, 1000)], 1, "q4"),
                             ([hb.r(w), hb.r(q)], 2, "binding"), ([hb.r(w), hb.r(q)], 0, "0 rows"),
                             ([hb.r(w), hb.r(w)], 1, "overlap|holds"), ([hb.r(w), hb.r(q)], 1 << 31, "too many")]:
        with pytest.raises(hb.HerbertError, match=match):
            gpu.launch(k, ranges, m)


def test_engine_choice_and_pins(hb, gpu):
    """The choice on the host: picks text, pinning it, and what a pin refuses."""
    w, x, y = matvec_bufs(hb, gpu, 128, 32, 2)
    y0 = np.arange(64, dtype=np.uint16)
    gpu.upload(y, y0)
    args = (128, 32, hb.Out.Residual, 32, 2, [hb.r(w)], hb.r(x), hb.r(y))
    with hb.Engine(gpu, "") as e:
        k = e.mv_q4(*args)
        assert gpu.kernel_kind(k) == hb.Kind.MATVEC_Q4
        assert np.array_equal(gpu.download(y, np.uint16, 64), y0)
        text = e.picks()
        with pytest.raises(hb.HerbertError, match="no weights"):
            e.mv_q4(128, 32, hb.Out.Bf16, 32, 2, [], hb.r(x), hb.r(y))
        with pytest.raises(hb.HerbertError, match="m <= 16"):
            e.mv_q4(128, 32, hb.Out.Bf16, 32, 17, [hb.r(w)], hb.r(x), hb.r(y))
        with pytest.raises(hb.HerbertError, match="0 rows"):
            e.mv_q4(128, 32, hb.Out.Bf16, 32, 0, [hb.r(w)], hb.r(x), hb.r(y))
        with pytest.raises(hb.HerbertError, match="group"):
            e.mv_q4(128, 32, hb.Out.Bf16, 0, 2, [hb.r(w)], hb.r(x), hb.r(y))
    with hb.Engine(None) as e:
        with pytest.raises(hb.HerbertError, match="without a context"):
            e.mv_q4(*args)
    with hb.Engine(gpu, "") as e:
        e.pin(text)
        assert e.mv_q4(*args) == k and e.picks() == text
        for bad in (text.replace(" m2", " m3"), text.replace("mv_q4\t", "mv_q5\t"), "mv_q4\tx\t-\t-\n"):
            with pytest.raises(hb.HerbertError, match="pin, line 1"):
                e.pin(bad)


@pytest.mark.parametrize("desc", [
    herbert_hip.matvec_q4(8, 1, herbert_hip.Out.Bf16),
    herbert_hip.matvec_q4(17408, 5120, herbert_hip.Out.F32, 32, 16, 64, 16, 16, 4),
    herbert_hip.matvec_q4(17408, 5120, herbert_hip.Out.Swiglu, 32, 16, 128, 16, 16, 1),
    herbert_hip.experts_q4(2048, 1024, herbert_hip.Out.Swiglu, 128, herbert_hip.Rows.Gather, 8, 256, 64),
    herbert_hip.q4_quantize(72, 3, 128), herbert_hip.q4_pack(72, 3, 64), herbert_hip.q4_dequantize(72, 3, 32),
    herbert_hip.block_norm(1, 1e-6), herbert_hip.block_norm(32768, 1e-6, True, True, True, herbert_hip.Gate.Elements, True),
])
def test_forms_compile(monkeypatch, desc):
    """By the compiler that the library loads, without a GPU."""
    monkeypatch.setenv("HB_CACHE_DIR", "")
    herbert_hip.check(herbert_hip.lib.hb_kernel_precompile(ctypes.byref(desc)))
