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


def limit(hb, gpu, desc, most, refusal="too many"):
    """A launch over `most` rows or matrices gets as far as its buffers' sizes, one more does not."""
    kern = gpu.pipeline(desc)
    b = [hb.r(gpu.alloc(64)), hb.r(gpu.alloc(64))]
    for call in (lambda m: gpu.launch(kern, b, m), lambda m: gpu.graph([hb.Op(kern, b, m)]), lambda m: gpu.time_ops([hb.Op(kern, b, m)])):
        with pytest.raises(hb.HerbertError) as e:
            call(most)
        assert refusal not in str(e.value) and "binding" in str(e.value), e.value
        with pytest.raises(hb.HerbertError, match=refusal):
            call(most + 1)


# Whole workgroups of 256 threads below 2^32 threads.
THREADS = 2 ** 32 - 256


@pytest.mark.parametrize("k", [16, 112, 128, 144, 2560, 17408, 1 << 20])
def test_grid_of_rows(hb, gpu, k):
    """Quantised rows take 16 threads a group of 128, read back one for 16 elements."""
    assert gpu.groups(gpu.pipeline(hb.f8_quantize_rows(k)), 1 << 12) * 256 >= 16 * -(-k // 128) << 12
    limit(hb, gpu, hb.f8_quantize_rows(k), THREADS // (16 * -(-k // 128)))
    if k > 16:  # of 16: one thread a row, more rows than m holds
        limit(hb, gpu, hb.f8_dequantize_rows(k), THREADS // (k // 16))


def test_rows_past_the_grid(hb, gpu):
    """80 GiB of rows, 1.25 2^32 threads."""
    kern = gpu.pipeline(hb.f8_quantize_rows(2560))
    with pytest.raises(hb.HerbertError, match="too many"):
        gpu.launch(kern, [hb.r(gpu.alloc(64)), hb.r(gpu.alloc(64))], 1 << 24)


@pytest.mark.parametrize("k,n", [(16, 1), (144, 130), (5120, 34816)])
def test_grid_of_matrices(hb, gpu, k, n):
    """A workgroup a block of 128 x 128; read back, a thread for 16 elements."""
    limit(hb, gpu, hb.f8_quantize(k, n), THREADS // (256 * -(-k // 128) * -(-n // 128)))
    if k * n > 16:
        limit(hb, gpu, hb.f8_dequantize(k, n), THREADS // (k // 16 * n))


def test_grid_of_routes(hb, gpu):
    """A wave a row, four of them a workgroup."""
    limit(hb, gpu, hb.route_topk(64, 4), THREADS // 64)


@pytest.mark.parametrize("k,n", [(64, 16), (2560, 18432)])
def test_grid_of_q4_matrices(hb, gpu, k, n):
    """A wave a tile, four of them a workgroup."""
    kern = gpu.pipeline(hb.q4_dequantize(k, n))
    per = gpu.groups(kern, 1 << 10) * 4 >> 10  # tiles a matrix
    limit(hb, gpu, hb.q4_dequantize(k, n), THREADS // (64 * per))
    with pytest.raises(hb.HerbertError, match="too many"):
        gpu.launch(kern, [hb.r(gpu.alloc(64)), hb.r(gpu.alloc(64))], 0xFFFFFFFF)


@pytest.mark.parametrize("out", ["Bf16", "F32", "Residual"])
@pytest.mark.parametrize("rows", [17, 64, 256, 1024])
def test_no_split(hb, gpu, out, rows):
    """ksplit 1 on a shape whose defaults split K: whole, and no workspace."""
    assert "_ks" in gpu.kernel_name(gpu.pipeline(hb.gemm_f8(9216, 2560, hb.Out[out], rows=rows)))
    whole = gpu.pipeline(hb.gemm_f8(9216, 2560, hb.Out[out], rows=rows, ksplit=1))
    assert "_ks" not in gpu.kernel_name(whole)
    size = 4 if out == "F32" else 2
    sizes = [16, hb.f8_bytes(9216, 2560), rows * hb.f8_row_bytes(9216), rows * 2560 * size]
    other = hb.Gpu(0)
    k = other.pipeline(hb.gemm_f8(9216, 2560, hb.Out[out], rows=rows, ksplit=1))
    b = [other.alloc(s) for s in sizes]
    held = hb.lib.fake_in_use()
    other.launch(k, [hb.r(v) for v in b + b[:1] * 2], rows)
    assert hb.lib.fake_in_use() == held
    other.close()
