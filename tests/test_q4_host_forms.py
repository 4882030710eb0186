"""What the library makes of 4-bit calls on the CPU, over a HIP runtime on host
memory: the fields a descriptor names are kept, kernels that do not belong
together are refused."""
import ctypes
import os
import subprocess

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


def experts(hb, **form):
    return hb.experts_q4(2048, 64, hb.Out.Bf16, 32, hb.Rows.Gather, 8, 64, 4, **form)


@pytest.mark.parametrize("form,name", [({}, "_r32_k4_w4_"), ({"split": 1}, "_k1_w4_"), ({"split": 4}, "_k4_w4_"),
                                       ({"split": 8}, "_k8_w8_"), ({"split": 16}, "_k16_w16_"), ({"waves": 2}, "_k2_w2_"),
                                       ({"waves": 8}, "_k4_w8_"), ({"split": 2, "waves": 8}, "_k2_w8_")])
def test_experts_fields_are_kept(hb, gpu, form, name):
    """A split that is named stays, with as many waves where those are left to
    the defaults; only a defaulted one yields to the waves."""
    assert name in gpu.kernel_name(gpu.pipeline(experts(hb, **form)))


@pytest.mark.parametrize("split,waves", [(8, 4), (16, 8), (2, 1)])
def test_experts_split_past_the_waves(hb, gpu, split, waves):
    """Refused, as the dense descriptor is, and not another order of sums."""
    for d in (experts(hb, split=split, waves=waves), hb.matvec_q4(2048, 64, hb.Out.Bf16, split=split, waves=waves)):
        with pytest.raises(hb.HerbertError, match="split no more"):
            gpu.pipeline(d)


@pytest.mark.parametrize("rows,split", [(32, 8), (64, 16), (128, 16)])
def test_experts_splits_compile(monkeypatch, rows, split):
    """By the compiler that the library loads, without a GPU."""
    monkeypatch.setenv("HB_CACHE_DIR", "")
    d = experts(herbert_hip, rows=rows, split=split, unroll=1)
    herbert_hip.check(herbert_hip.lib.hb_kernel_precompile(ctypes.byref(d)))


def pin_text(hb, gpu, desc):
    return "%s\t%s" % (gpu.kernel_name(gpu.pipeline(desc)), " ".join(str(getattr(desc, f)) for f in hb._DESC_FIELDS))


def test_pins_of_bf16_choices_take_no_4bit_kernel(hb, gpu):
    """A 4-bit kernel binds as much as its bf16 counterpart, so only the pin can
    tell that it would read bf16 weights as codes."""
    mv = hb.matvec(2048, 64, hb.Out.Bf16)
    mv_q4 = hb.matvec_q4(2048, 64, hb.Out.Bf16)
    sort = hb.Desc(kind=hb.Kind.SORT, experts=64, top_k=8, bm=16, rows_max=4)
    tile = dict(top_k=8, experts=64, bm=16, tiles=hb.moe_tiles(4, 8, 64, 16), wm=1, wn=4, bn=128, bk=64, rows_max=4)
    gu = hb.gemm_mma_rows(2048, 1024, hb.Out.Bf16, rows_of=hb.Rows.Gather, **tile)
    dn = hb.gemm_mma_rows(512, 2048, hb.Out.Bf16, rows_of=hb.Rows.Scatter, **tile)
    gu_q4 = hb.experts_q4(2048, 1024, hb.Out.Swiglu, 32, hb.Rows.Gather, 8, 64, 4)
    dn_q4 = hb.experts_q4(512, 2048, hb.Out.Bf16, 32, hb.Rows.Scatter, 8, 64, 4)

    def line(*descs):
        return "experts\tkey\t16\t%s\t-\t-\n" % "\t".join(pin_text(hb, gpu, d) for d in descs)

    with hb.Engine(gpu, "") as e:
        good = "mv\t2048x64 Bf16 m1\t%s\n" % pin_text(hb, gpu, mv) + line(sort, gu, dn)
        e.pin(good)
        text = e.picks()
        assert [gpu.kernel_name(gpu.pipeline(d)) in text for d in (mv, sort, gu, dn)] == [True] * 4
        with pytest.raises(hb.HerbertError, match="no matvec kernel"):
            e.pin("mv\t2048x64 Bf16 m1\t%s\n" % pin_text(hb, gpu, mv_q4))
        for descs in ((sort, gu_q4, dn_q4), (sort, gu_q4, dn), (sort, gu, dn_q4)):
            with pytest.raises(hb.HerbertError, match="no grouped GEMM"):
                e.pin(line(*descs))
        assert e.picks() == text


def test_experts_run_takes_no_swiglu_down(hb, gpu):
    """A down kernel of Out::Swiglu writes rows of half its W rows."""
    E, K, H, MI, rows = 64, 4, 256, 128, 8
    wg, wd = gpu.alloc(E * hb.q4_bytes(H, 2 * MI)), gpu.alloc(E * hb.q4_bytes(MI, H))
    with hb.Engine(gpu, "") as e:
        layer = hb.MoeLayer(gpu, e, E, K, H, MI, rows, wg, wd, q4_group=32)

    def run():
        return hb.lib.hb_moe_experts_run(gpu.h, (ctypes.c_int32 * 4)(*layer.kernels), layer.swiglu_k, layer.combine_k,
                                         ctypes.byref(layer.io), hb.r(layer.buf["out"]), rows)

    assert run() == 0, hb.last_error()
    layer.kernels[2] = gpu.pipeline(hb.experts_q4(MI, H, hb.Out.Swiglu, 32, hb.Rows.Scatter, K, E, rows))
    assert run() == hb.ERR_INVALID and "down" in hb.last_error()


def test_a_range_past_64_bits_is_refused(hb, gpu):
    """An offset and a size whose sum wraps lie outside the buffer, however
    small the sum is."""
    k = gpu.pipeline(hb.matvec_q4(128, 32, hb.Out.F32, mv_m=1))
    w, x, y = gpu.alloc(hb.q4_bytes(128, 32)), gpu.alloc(256), gpu.alloc(128)
    gpu.launch(k, [hb.r(w), hb.r(x), hb.r(y)], 1)
    for bad in (hb.r(y, 4, 2 ** 64 - 4), hb.r(y, 64, 2 ** 64 - 32), hb.r(y, 0, 129), hb.r(y, 129)):
        with pytest.raises(hb.HerbertError, match="outside buffer"):
            gpu.launch(k, [hb.r(w), hb.r(x), bad], 1)


def test_native_host_counts_its_bytes(hb, tmp_path):
    """hb_gemm over the host runtime, whose launches take 10 us each: GB/s of
    weights, x and y in each Out, four bytes an f32."""
    lib = os.path.dirname(hb.LIB_PATH)
    exe = str(tmp_path / "hb_gemm")
    subprocess.run(["g++", "-O1", "-std=c++17", os.path.join(host_gpu.PKG, "csrc", "hb_cli.cpp"), "-I", os.path.join(host_gpu.ROOT, "include"),
                    "-L", lib, "-lherbert_hip", "-Wl,-rpath," + lib, "-o", exe], check=True)
    r = subprocess.run([exe, "--reps", "2", "mv:16x64x4096", "mv:16x64x4096f", "mv:16x64x4096r"],
                       capture_output=True, text=True, timeout=60, env=dict(os.environ, HB_CACHE_DIR=""))
    assert r.returncode == 0, r.stderr
    y, x, w = 16 * 4096, 2 * 16 * 64, 2 * 64 * 4096
    want = [w + x + 2 * y, w + x + 4 * y, w + x + 4 * y]
    assert [line.split()[-2] for line in r.stdout.splitlines()] == ["%.1f" % (b / 1e4) for b in want], r.stdout
