"""The 8-bit kernels' forms and launches on the CPU over a HIP runtime on host
memory: forms that are refused, grids at their limit, what a split of K takes of
the workspace, and which forms the defaults take."""
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


def chunks(waves, rows):
    """Per row of an operand's stage, the chunk of K that each of its eight LDS
    places holds, as a workgroup of `waves` waves loads it: lane l of a wave loads
    rows wave * 8 + l / 8 + 8 waves i, always the chunk that its first row's
    swizzle puts at place l % 8."""
    held = {}
    for wave in range(waves):
        for lane in range(64):
            first = wave * 8 + lane // 8
            for row in range(first, rows, 8 * waves):
                held.setdefault(row, {})[lane % 8] = lane % 8 ^ (first >> 1 & 7)
    return held


@pytest.mark.parametrize("waves", range(1, 17))
def test_swizzle_of_a_waves_loads(waves):
    """A fragment reads chunk c of a row at place c ^ (row >> 1): the place that
    holds it for every row where the waves are even in number, and no others are
    taken."""
    held = chunks(waves, 256)
    wrong = sum(held[row][c ^ (row >> 1 & 7)] != c for row in held for c in range(8))
    assert (wrong == 0) == (waves % 2 == 0)


@pytest.mark.parametrize("tile", [dict(bm=32, bn=32, wm=1, wn=1), dict(bm=32, bn=96, wm=1, wn=3), dict(bm=64, bn=160, wm=1, wn=5),
                                  dict(bm=64, bn=224, wm=1, wn=7), dict(bm=64, wn=1)])
@pytest.mark.parametrize("out", ["Bf16", "F32", "Residual"])
def test_odd_waves_refused(hb, gpu, tile, out):
    with pytest.raises(hb.HerbertError, match="even number of waves"):
        gpu.pipeline(hb.gemm_f8(256, 512, hb.Out[out], **tile))


@pytest.mark.parametrize("bm", [32, 64])
def test_odd_waves_of_experts_refused(hb, gpu, bm):
    with pytest.raises(hb.HerbertError, match="even number of waves"):
        gpu.pipeline(hb.experts_f8(256, 512, hb.Out.Bf16, hb.Rows.Gather, 2, 8, 64, bm, wm=1, wn=1, bn=32))
