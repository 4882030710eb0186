"""What the library makes of 4-bit calls on the CPU, over a HIP runtime on host
memory: the fields a descriptor names are kept, kernels that do not belong
together are refused."""
import ctypes

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
