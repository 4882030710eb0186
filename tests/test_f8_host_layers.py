"""The layers over 8-bit experts and their routes on the CPU, over a HIP runtime
on host memory: what a refused one leaves behind, what a layer allocates."""
import ctypes

import numpy as np
import pytest

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


E, K = 64, 4  # route_qwen takes experts by 64


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("kw", [dict(hidden=264), dict(hidden=100), dict(inter=64), dict(route=lambda hb: hb.route_topk(E, K, groups=5)),
                                dict(route=lambda hb: hb.route_topk(E, K + 1)), dict(route=lambda hb: hb.route_topk(E, K, bias=True)),
                                dict(q4_group=32)])
def test_refused_layer(hb, gpu, rows, kw):
    """A MoeLayer, and a MoeBlock around it, that are refused hold no memory."""
    kw = dict(kw)
    h, mi = kw.pop("hidden", 256), kw.pop("inter", 128)
    if "route" in kw:
        kw["route"] = kw["route"](hb)
    w = gpu.alloc(64)
    held = hb.lib.fake_in_use()
    with pytest.raises(hb.HerbertError):
        hb.MoeLayer(gpu, None, E, K, h, mi, rows, w, w, f8=True, **kw)
    assert hb.lib.fake_in_use() == held
    names = {n: w for n in ("post_norm", "router", "w_gate_up", "w_down", "s_gate_up", "s_down", "shared_gate")}
    names["route_bias"] = None
    with pytest.raises(hb.HerbertError):
        hb.MoeBlock(gpu, None, E, K, h, mi, 128, rows, names, np.zeros((rows, h), np.uint16), f8=True, **kw)
    assert hb.lib.fake_in_use() == held


class NoWeights:
    """A checkpoint whose reading would be one too many."""

    def has(self, key):
        return False

    def upload(self, *a):
        raise AssertionError("uploaded")

    upload_f8 = upload


@pytest.mark.parametrize("hidden,inter", [(264, 128), (256, 64), (256, 200)])
def test_refused_mlp(hb, gpu, hidden, inter):
    with hb.Engine(gpu, "prefill.block=128") as e:
        held = hb.lib.fake_in_use()
        with pytest.raises(hb.HerbertError):
            hb.PrefillMlp(gpu, e, NoWeights(), 0, hidden, inter, f8=True)
        assert hb.lib.fake_in_use() == held


@pytest.mark.parametrize("rows,bm", [(1, 16), (40, 32), (1000, 128)])
def test_layer_memory(hb, gpu, rows, bm):
    """An 8-bit layer's buffers are those its launches bind: no gate and up rows, x's quantised rows
    only where a kernel writes them."""
    h, mi, pairs = 256, 128, rows * K
    w = gpu.alloc(E * hb.f8_bytes(h, 2 * mi)), gpu.alloc(E * hb.f8_bytes(mi, h))
    held = hb.lib.fake_in_use()
    layer = hb.MoeLayer(gpu, None, E, K, h, mi, rows, *w, f8=True)
    assert layer.bm == bm
    want = {"state": 16, "scores": rows * E * 2, "route": rows * 8 * K, "list": pairs * 4, "tiles": (1 + 3 * hb.moe_tiles(rows, K, E, 16)) * 4,
            "x": rows * h * 2, "ehb": pairs * (2 * mi if bm == 16 else hb.f8_row_bytes(mi)), "ey": pairs * h * 2, "out": rows * h * 2}
    if bm > 16:
        want["xs"] = rows * hb.f8_row_bytes(h)
    assert {n: gpu.size(b) for n, b in layer.buf.items() if n not in ("w_gate_up", "w_down")} == want
    assert hb.lib.fake_in_use() - held == sum(-(-v // 256) * 256 for v in want.values())  # each a multiple of 256
    names = [gpu.kernel_name(op.kernel) for op in layer.ops()]
    assert len(names) == (6 if bm > 16 else 5) and not any("swiglu" in n for n in names)
    layer.free()
    assert hb.lib.fake_in_use() == held


@pytest.mark.parametrize("f32", [False, True])
def test_scores_of_another_type(hb, gpu, f32):
    """bf16 scores where the route reads f32 would fill half of the buffer, f32 ones be read as bf16."""
    w = gpu.alloc(64)
    held = hb.lib.fake_in_use()
    scores = np.zeros((4, E), np.uint16 if f32 else np.float32)
    with pytest.raises(hb.HerbertError, match="scores in %s" % ("f32" if f32 else "bf16")):
        hb.MoeLayer(gpu, None, E, K, 256, 128, 4, w, w, f8=True, scores=scores, route=hb.route_topk(E, K, f32=f32))
    assert hb.lib.fake_in_use() == held


@pytest.mark.parametrize("rows", [2, 40])
def test_kernels_of_another_layer(hb, gpu, rows):
    """hb_moe_experts_run refuses 8-bit kernels whose sizes, experts or top_k differ: h would be read as
    rows of another length, or experts' rows be left unwritten."""
    h, mi = 256, 128
    w = gpu.alloc(2 * E * hb.f8_bytes(h, 4 * mi)), gpu.alloc(2 * E * hb.f8_bytes(2 * mi, h))
    layer = hb.MoeLayer(gpu, None, E, K, h, mi, rows, *w, f8=True)
    sort, gu, dn, quantize = layer.kernels

    def experts(kdim, n, gate_up, top_k=K, count=E):
        out, of = (hb.Out.Swiglu, hb.Rows.Gather) if gate_up else (hb.Out.Bf16, hb.Rows.Scatter)
        return gpu.pipeline(hb.experts_f8(kdim, n, out, of, top_k, count, rows, layer.bm))

    def sorted_by(top_k, count):
        return gpu.pipeline(hb.Desc(kind=hb.Kind.SORT, experts=count, top_k=top_k, bm=layer.bm, rows_max=rows))

    for ks in ([sort, experts(h, 4 * mi, True), dn, quantize], [sort, gu, experts(2 * mi, h, False), quantize],
               [sort, gu, experts(mi, 2 * h, False), quantize], [sort, experts(h, 2 * mi, True, K // 2), dn, quantize],
               [sort, gu, experts(mi, h, False, K // 2), quantize], [sort, experts(h, 2 * mi, True, K, E // 2), dn, quantize],
               [sort, gu, experts(mi, h, False, K, 2 * E), quantize], [sorted_by(K, 2 * E), gu, dn, quantize],
               [sorted_by(K // 2, E), gu, dn, quantize]):
        hb.lib.fake_forget()
        rc = hb.lib.hb_moe_experts_run(gpu.h, (ctypes.c_int32 * 4)(*ks), layer.swiglu_k, layer.combine_k, ctypes.byref(layer.io),
                                       hb.r(layer.buf["out"]), rows)
        assert rc == hb.ERR_INVALID and "moe experts in 8 bits" in hb.last_error(), ks
        assert hb.lib.fake_launches() == 0
