"""What the library refuses of the 8-bit kernels and route_topk, on the CPU over
a HIP runtime on host memory, and the forms that compile."""
import ctypes

import numpy as np
import pytest

import f8_ref as f8
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


def test_bytes(hb):
    assert hb.f8_row_bytes(16) == 128 and hb.f8_row_bytes(512) == 640 and hb.f8_row_bytes(2560) == 2688 and hb.f8_row_bytes(112) == 128
    assert hb.f8_bytes(16, 1) == 32 and hb.f8_bytes(128, 128) == 16400 and hb.f8_bytes(2560, 10240) == 2560 * 10240 + 4 * 20 * 80
    assert hb.f8_bytes(1 << 20, 1 << 24) == (1 << 44) + (1 << 32)
    for k, n in [(0, 1), (16, 0), (24, 1), (8, 1), ((1 << 20) + 16, 1), (16, (1 << 24) + 1)]:
        with pytest.raises(hb.HerbertError):
            hb.f8_bytes(k, n)
    for k in (0, 8, 100):
        with pytest.raises(hb.HerbertError):
            hb.f8_row_bytes(k)


def test_tile_rows(hb):
    """A power of two of 16 to 128 that grows with the rows an expert has."""
    last = 0
    for rows in (1, 8, 64, 128, 500, 1000, 2048, 8192, 1 << 20, 0xFFFFFFFF):
        bm = hb.f8_tile_rows(rows, 8, 256)
        assert bm in (16, 32, 64, 128) and bm >= last
        last = bm
    assert hb.f8_tile_rows(1, 8, 256) == 16 and last == 128


def test_reference_codes():
    """The tests' own e4m3: codes of all values are themselves, ties go to even codes."""
    c = np.arange(256)
    c = c[(c & 127) != 127]
    back = f8.encode(f8.VALUES[c])
    assert np.array_equal(f8.VALUES[back], f8.VALUES[c]) and (back[c != 128] == c[c != 128]).all()
    mid = (f8.VALUES[:126] + f8.VALUES[1:127]) / 2
    assert np.array_equal(f8.encode(mid), np.arange(126) + np.arange(126) % 2)
    assert f8.encode(np.array([np.nan, 464.0, -448.0])).tolist() == [0x7F, 126, 254]


@pytest.mark.parametrize("make,match", [
    (lambda hb: hb.f8_quantize(100, 16), "K a multiple of 16"),
    (lambda hb: hb.f8_quantize(16, 0), "N up to"),
    (lambda hb: hb.f8_quantize_rows(8), "K a multiple of 16"),
    (lambda hb: hb.f8_dequantize((1 << 20) + 16, 1), "up to 2\\^20"),
    (lambda hb: hb.f8_dequantize(16, (1 << 24) + 1), "up to 2\\^24"),
    (lambda hb: hb.f8_quantize_rows(16).replace(form=2), "a matrix or rows"),
    (lambda hb: hb.matvec_f8(100, 16, hb.Out.Bf16), "K a multiple of 16"),
    (lambda hb: hb.matvec_f8(128, 16, hb.Out.Bf16, mv_m=17), "m <= 16"),
    (lambda hb: hb.matvec_f8(128, 16, 4), "out"),
    (lambda hb: hb.matvec_f8(128, 128, hb.Out.Swiglu), "multiple of 128"),
    (lambda hb: hb.matvec_f8(128, 256, hb.Out.Swiglu, rows=16), "rows a wave"),
    (lambda hb: hb.matvec_f8(128, 64, hb.Out.Bf16, rows=128), "rows a wave"),
    (lambda hb: hb.Desc(kind=hb.Kind.GEMM_F8, k=128, n=64, out=hb.Out.Bf16, mfma=32), "16 a wave"),
    (lambda hb: hb.matvec_f8(128, 64, hb.Out.Bf16, waves=3), "waves"),
    (lambda hb: hb.matvec_f8(128, 64, hb.Out.Bf16, split=8, waves=4), "split"),
    (lambda hb: hb.matvec_f8(128, 64, hb.Out.Bf16, unroll=5), "unroll"),
    (lambda hb: hb.matvec_f8(4096, 64, hb.Out.Bf16, mv_m=16, rows=64, split=16, waves=16, unroll=1), "stages"),
    (lambda hb: hb.experts_f8(128, 64, hb.Out.F32, hb.Rows.Gather, 8, 64, 4, 16), "bf16 out"),
    (lambda hb: hb.experts_f8(128, 64, hb.Out.F32, hb.Rows.Gather, 8, 64, 4, 64), "bf16 out"),
    (lambda hb: hb.experts_f8(128, 64, hb.Out.Bf16, hb.Rows.Sorted, 8, 64, 4, 16), "rows_of"),
    (lambda hb: hb.experts_f8(128, 64, hb.Out.Bf16, hb.Rows.Sorted, 8, 64, 4, 64), "rows_of"),
    (lambda hb: hb.experts_f8(128, 64, hb.Out.Bf16, hb.Rows.Gather, 8, 64, 4, 64).replace(tiles=0), "tiles"),
    (lambda hb: hb.experts_f8(128, 64, hb.Out.Bf16, hb.Rows.Gather, 8, 2048, 4, 64), "experts"),
    (lambda hb: hb.experts_f8(128, 64, hb.Out.Bf16, hb.Rows.Gather, 8, 4, 4, 64), "top_k"),
    (lambda hb: hb.experts_f8(128, 64, hb.Out.Bf16, hb.Rows.Gather, 8, 64, 1 << 26, 64), "pairs"),
    (lambda hb: hb.experts_f8(128, 256, hb.Out.Swiglu, hb.Rows.Scatter, 8, 64, 4, 64), "no scatter"),
    (lambda hb: hb.gemm_f8(136, 64, hb.Out.Bf16), "K a multiple of 16"),
    (lambda hb: hb.gemm_f8(65552, 64, hb.Out.Bf16), "up to 2\\^16"),
    (lambda hb: hb.gemm_f8(65536, 32768, hb.Out.Bf16), "below 2\\^31"),
    (lambda hb: hb.gemm_f8(128, 384, hb.Out.Swiglu), "multiple of 128"),
    (lambda hb: hb.gemm_f8(128, 512, hb.Out.Swiglu, bn=128), "tiles"),
    (lambda hb: hb.gemm_f8(128, 64, hb.Out.Bf16, bm=48), "tiles"),
    (lambda hb: hb.gemm_f8(128, 64, hb.Out.Bf16, bm=16), "tiles"),
    (lambda hb: hb.gemm_f8(128, 64, hb.Out.Bf16, bm=512), "tiles"),
    (lambda hb: hb.gemm_f8(128, 64, hb.Out.Bf16, bn=288), "tiles"),
    (lambda hb: hb.gemm_f8(128, 64, hb.Out.Bf16, bn=48), "tiles"),
    (lambda hb: hb.gemm_f8(128, 64, hb.Out.Bf16, bm=64, wm=8), "tiles"),
    (lambda hb: hb.gemm_f8(128, 64, hb.Out.Bf16, bm=256, bn=256, stages=3), "stages within"),
    (lambda hb: hb.gemm_f8(128, 64, hb.Out.Bf16, stages=5), "stages"),
    (lambda hb: hb.gemm_f8(128, 64, hb.Out.Bf16, ksplit=2), "split K"),
    (lambda hb: hb.gemm_f8(4096, 66, hb.Out.Bf16, ksplit=17), "split K"),
    (lambda hb: hb.gemm_f8(4096, 256, hb.Out.Swiglu, ksplit=2), "split K"),
    (lambda hb: hb.gemm_f8(128, 64, 4), "out"),
    (lambda hb: hb.route_topk(0, 1), "1 to 1024"),
    (lambda hb: hb.route_topk(1025, 1), "1 to 1024"),
    (lambda hb: hb.route_topk(64, 33), "1 to 32"),
    (lambda hb: hb.route_topk(64, 0), "1 to 32"),
    (lambda hb: hb.route_topk(4, 5), "no more than their experts"),
    (lambda hb: hb.route_topk(64, 5, groups=5), "groups of equal size"),
    (lambda hb: hb.route_topk(130, 1, groups=65), "up to 64 groups"),
    (lambda hb: hb.route_topk(64, 9, groups=8, top_groups=1), "no more than their experts"),
    (lambda hb: hb.route_topk(64, 4, groups=8, top_groups=9), "groups"),
    (lambda hb: hb.route_topk(64, 4).replace(form=32), "parts"),
    (lambda hb: hb.route_topk(64, 4, group_top=3), "one or two"),
    (lambda hb: hb.route_topk(64, 4, scale=0.0), "scale of 0"),
])
def test_refused_descriptors(hb, gpu, make, match):
    with pytest.raises(hb.HerbertError, match=match):
        gpu.pipeline(make(hb))


def refused(hb, gpu, k, good, m, cases):
    """`good` is launched (the fake runtime's launches have three bindings or more); each (changed
    ranges, m, match) is refused by launch, graph and time_ops."""
    if len(good) > 2:
        gpu.launch(k, good, m)
    for over, rows, match in cases:
        ranges = [over.get(i, v) for i, v in enumerate(good)] if isinstance(over, dict) else over
        for call in (lambda: gpu.launch(k, ranges, rows), lambda: gpu.graph([hb.Op(k, ranges, rows)]),
                     lambda: gpu.time_ops([hb.Op(k, ranges, rows)])):
            with pytest.raises(hb.HerbertError, match=match):
                call()


def test_refused_launches(hb, gpu):
    R = hb.r
    x, y = gpu.alloc(3 * 144 * 2 + 64), gpu.alloc(3 * 256 + 64)
    refused(hb, gpu, gpu.pipeline(hb.f8_quantize_rows(144)), [R(x, 2), R(y)], 3, [
        ({0: R(x, 1)}, 3, "multiple of 2"), ({1: R(y, 8)}, 3, "multiple of 16"), ({0: R(x, 0, 862)}, 3, "binding 0"),
        ({1: R(y, 0, 767)}, 3, "binding 1"), ({1: R(x)}, 1, "overlap"), ({}, 0, "0 rows"), ([R(x)], 1, "bindings"),
        ({}, 1 << 31, "too many|holds")])
    refused(hb, gpu, gpu.pipeline(hb.f8_dequantize_rows(144)), [R(y), R(x)], 3, [
        ({1: R(x, 0, 862)}, 3, "binding 1"), ({0: R(y, 0, 767)}, 3, "binding 0"), ({1: R(y, 2)}, 1, "overlap")])
    w, q = gpu.alloc(2 * 130 * 144 * 2), gpu.alloc(2 * hb.f8_bytes(144, 130))
    refused(hb, gpu, gpu.pipeline(hb.f8_quantize(144, 130)), [R(w), R(q)], 2, [
        ({0: R(w, 2)}, 2, "binding 0"), ({1: R(q, 16)}, 2, "binding 1"), ({}, 3, "binding"), ({}, 0, "0 rows"),
        ({}, 0xFFFFFFFF, "too many|holds")])
    big = gpu.pipeline(hb.f8_dequantize(1 << 20, 1 << 24))
    with pytest.raises(hb.HerbertError, match="too many"):
        gpu.launch(big, [R(q), R(w)], 1)


def test_refused_matvec_launches(hb, gpu):
    R = hb.r
    w, x, y = gpu.alloc(hb.f8_bytes(128, 32) + 32), gpu.alloc(2 * 256 + 64), gpu.alloc(2 * 128 + 64)
    refused(hb, gpu, gpu.pipeline(hb.matvec_f8(128, 32, hb.Out.F32, mv_m=2)), [R(w), R(x, 16), R(y, 4)], 2, [
        ({}, 0, "0 rows"), ({}, 3, "rows: 1..2"), ({0: R(w, 0, hb.f8_bytes(128, 32) - 1)}, 1, "binding 0"), ({0: R(w, 8)}, 1, "multiple of 16"),
        ({1: R(x, 0, 511)}, 2, "binding 1"), ({2: R(y, 0, 255)}, 2, "binding 2"), ({1: R(x, 2)}, 1, "multiple of 16"),
        ({2: R(y, 2)}, 1, "multiple of 4"), ({2: R(x, 4)}, 1, "overlap"), ({2: R(w, 1024)}, 1, "overlap")])


def test_refused_gemm_launches(hb, gpu):
    R = hb.r
    m, k, n = 3, 144, 512
    st, w, x = gpu.alloc(16), gpu.alloc(hb.f8_bytes(k, n)), gpu.alloc(m * hb.f8_row_bytes(k) + 64)
    y = gpu.alloc(m * n * 4 + 64)
    bad = [({}, 0, "0 rows"), ({0: R(st, 0, 12)}, m, "binding 0"), ({1: R(w, 0, hb.f8_bytes(k, n) - 1)}, m, "binding 1"),
           ({2: R(x, 0, m * hb.f8_row_bytes(k) - 1)}, m, "binding 2"), ({2: R(x, 4)}, m, "multiple of 16"), ({3: R(w, 16)}, m, "overlap"),
           ({}, 1 << 24, "2 GiB|holds")]
    for out, size, align in [(hb.Out.Bf16, n * 2, 2), (hb.Out.F32, n * 4, 4), (hb.Out.Swiglu, hb.f8_row_bytes(n // 2), 16)]:
        kern = gpu.pipeline(hb.gemm_f8(k, n, out))
        refused(hb, gpu, kern, [R(st), R(w), R(x), R(y), R(st), R(st)], m, bad + [
            ({3: R(y, 0, m * size - 1)}, m, "binding 3"), ({3: R(y, align // 2)}, m, "multiple of %d" % align)])


@pytest.mark.parametrize("bm", [16, 64])
def test_refused_experts_launches(hb, gpu, bm):
    t, top_k, experts, k, n = 4, 2, 16, 128, 256
    kern = gpu.pipeline(hb.experts_f8(k, n, hb.Out.Swiglu, hb.Rows.Gather, top_k, experts, t, bm))
    assert gpu.groups(kern, 1) <= 16 and gpu.groups(kern, t) <= 64
    rows = bm == 16
    sizes = [16, experts * hb.f8_bytes(k, n), t * (2 * k if rows else hb.f8_row_bytes(k)),
             t * top_k * (n if rows else hb.f8_row_bytes(n // 2)), t * top_k * 4, (1 + 3 * hb.moe_tiles(t, top_k, experts, bm)) * 4]
    b = [gpu.alloc(s) for s in sizes]
    refused(hb, gpu, kern, [hb.r(x) for x in b], t, [({i: hb.r(b[i], 0, s - 1)}, t, "binding %d" % i) for i, s in enumerate(sizes)] +
            [({}, t + 1, "rows_max")])


def test_refused_route_launches(hb, gpu):
    R = hb.r
    m, e, k = 3, 40, 4
    s, o, b = gpu.alloc(m * e * 4 + 64), gpu.alloc(m * k * 8 + 64), gpu.alloc(e * 4 + 8)
    for f32, size in ((False, 2), (True, 4)):
        kern = gpu.pipeline(hb.route_topk(e, k, bias=True, f32=f32))
        refused(hb, gpu, kern, [R(s, size), R(o, 4), R(b)], m, [
            ({}, 0, "0 rows"), ({0: R(s, 0, m * e * size - 1)}, m, "binding 0"), ({0: R(s, size // 2)}, m, "multiple of %d" % size),
            ({1: R(o, 0, m * k * 8 - 1)}, m, "binding 1"), ({1: R(o, 2)}, m, "multiple of 4"), ({2: R(b, 0, e * 4 - 1)}, m, "binding 2"),
            ({2: R(b, 2)}, m, "multiple of 4"), ({1: R(s, 16)}, m, "overlap"), ([R(s), R(o)], m, "bindings"),
            ({}, 1 << 26, "too many")])


@pytest.mark.parametrize("desc", [
    herbert_hip.f8_quantize_rows(16), herbert_hip.f8_quantize(144, 1), herbert_hip.f8_dequantize_rows(17408), herbert_hip.f8_dequantize(16, 300),
    herbert_hip.matvec_f8(16, 1, herbert_hip.Out.Bf16), herbert_hip.matvec_f8(17408, 5120, herbert_hip.Out.F32, 16, 64, 4, 4, 2),
    herbert_hip.matvec_f8(2560, 18432, herbert_hip.Out.Swiglu, 16, 64, 8, 8, 1),
    herbert_hip.experts_f8(2048, 1024, herbert_hip.Out.Swiglu, herbert_hip.Rows.Gather, 8, 256, 64, 16),
    herbert_hip.experts_f8(2048, 1024, herbert_hip.Out.Swiglu, herbert_hip.Rows.Gather, 8, 256, 4096, 128),
    herbert_hip.experts_f8(512, 2048, herbert_hip.Out.Bf16, herbert_hip.Rows.Scatter, 8, 256, 4096, 32),
    herbert_hip.gemm_f8(16, 1, herbert_hip.Out.Bf16), herbert_hip.gemm_f8(65536, 16384, herbert_hip.Out.F32, bm=256, bn=128),
    herbert_hip.route_topk(1, 1), herbert_hip.route_topk(1024, 32, herbert_hip.Score.Sigmoid, True, 64, 3, 2, False, -1.5, True),
])
def test_forms_compile(monkeypatch, desc):
    """By the compiler that the library loads, without a GPU."""
    monkeypatch.setenv("HB_CACHE_DIR", "")
    herbert_hip.check(herbert_hip.lib.hb_kernel_precompile(ctypes.byref(desc)))
