"""The 8-bit kernels' forms and launches on the CPU over a HIP runtime on host
memory: forms that are refused, grids at their limit, what a split of K takes of
the workspace, and which forms the defaults take."""
import math
import random
import re

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


class Down:
    """A context with a down product of up to 1024 rows, whose defaults split K, and its buffers."""
    K, N, ROWS = 9216, 2560, (128, 256, 512, 1024)

    def __init__(self, hb):
        self.hb, self.g = hb, hb.Gpu(0)
        sizes = [16, hb.f8_bytes(self.K, self.N), 1024 * hb.f8_row_bytes(self.K), 1024 * self.N * 2]
        b = [hb.r(self.g.alloc(s)) for s in sizes]
        self.bind = b + b[:1] * 2

    def build(self, rows, **form):
        return self.g.pipeline(self.hb.gemm_f8(self.K, self.N, self.hb.Out.Residual, rows=rows, **form))

    def graph(self, kern, rows):
        return self.g.graph([self.hb.Op(kern, self.bind, rows)])

    def close(self):
        self.hb.lib.fake_limit(2 ** 64 - 1)
        self.g.close()


@pytest.fixture()
def down(hb):
    d = Down(hb)
    yield d
    d.close()


def test_workspace_when_built(hb, down):
    """Kernels of every bucket, a graph of the shortest one's, the others' launches beside it: the
    building made their room, no launch allocates."""
    kern = {m: down.build(m) for m in down.ROWS}
    assert all("_ks" in down.g.kernel_name(k) for k in kern.values())
    tries = hb.lib.fake_malloc_tries()
    graph = down.graph(kern[128], 128)
    for m in down.ROWS:
        down.g.launch(kern[m], down.bind, m)
    graph.launch()
    assert hb.lib.fake_malloc_tries() == tries
    graph.free()


def test_same_form_for_more_rows(hb, down):
    """A kernel that is there already, built again for more rows, makes their room too."""
    form = dict(bm=128, bn=128, ksplit=2)
    kern = down.build(128, **form)
    assert down.build(1024, **form) == kern
    graph = down.graph(kern, 128)
    down.g.launch(kern, down.bind, 1024)
    graph.free()


def test_built_beside_a_graph(hb, down):
    """A recorded graph holds the workspace: the defaults' product for more rows is unsplit and runs,
    a split that the caller named is refused at its launch, and after the graph both split."""
    small = down.build(128)
    graph = down.graph(small, 64)
    whole = down.build(1024)
    assert "_ks" not in down.g.kernel_name(whole)
    down.g.launch(whole, down.bind, 1024)
    named = down.build(1024, bm=128, bn=128, ksplit=8)
    with pytest.raises(hb.HerbertError, match="recorded graph"):
        down.g.launch(named, down.bind, 1024)
    graph.free()
    assert "_ks" in down.g.kernel_name(down.build(1024))
    down.g.launch(named, down.bind, 1024)


def test_built_without_memory(hb, down):
    """No memory for the slabs: unsplit, and as much in use as before."""
    held = hb.lib.fake_in_use()
    hb.lib.fake_limit(held + (1 << 20))
    kern = down.build(1024)
    assert "_ks" not in down.g.kernel_name(kern) and hb.lib.fake_in_use() == held
    down.g.launch(kern, down.bind, 1024)


def test_no_rows_named(hb, down):
    """Without rows the product is built for 2048, its workspace too."""
    kern = down.g.pipeline(hb.gemm_f8(17408, 1024, hb.Out.Bf16))
    assert "_ks" in down.g.kernel_name(kern)
    assert hb.lib.fake_in_use() > 2 * 2048 * 1024 * 4


@pytest.mark.parametrize("score", [2, 4, -1, 3.5])
def test_unknown_score_refused(hb, score):
    """A score that is none would set another of the descriptor's parts, a bias's binding for one."""
    with pytest.raises(hb.HerbertError, match="softmax or sigmoid"):
        hb.route_topk(64, 4, score=score)
    assert hb.route_topk(64, 4, score=hb.Score.Sigmoid).form & 1 and not hb.route_topk(64, 4, score=hb.Score.Softmax).form & 1


def test_defaults_are_tested(hb, gpu):
    """Every form that the defaults take, over the shapes from one row and 16 K to long prompts of the
    largest matrices, is one that the GPU tests run; and they take all of those."""
    import test_gpu_f8_forms as forms

    def tag(f):
        return "_t%dx%d_w%dx%d_d%d_b4%s" % (f["bn"], f["bm"], f["wn"], f["wm"], f["stages"] - 1, "_fa" if f["sched"] else "")

    tested = {"sw": forms.SWIGLU, "f32": forms.F32, "bf16": forms.DENSE, "res": forms.DENSE}
    tested = {out: {tag(f) for f in fs} for out, fs in tested.items()}
    taken = {out: set() for out in tested}
    rng = random.Random(5)

    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    for _ in range(3000):
        out = rng.choice(list(hb.Out))
        n = 256 * size(1, 136) if out == hb.Out.Swiglu else size(16, 34816)
        name = gpu.kernel_name(gpu.pipeline(hb.gemm_f8(16 * size(1, 1088), n, out, rows=size(1, 8192))))
        kind, form, parts = re.search(r"gemm_f8_\d+x\d+_(sw|f32|bf16|res)(_t.*?)(_ks\d)?$", name).groups()
        assert form in tested[kind] and parts in (None, "_ks2", "_ks4", "_ks8"), name
        taken[kind].add(form)
    assert taken == tested


@pytest.mark.parametrize("hidden,inter", [(400, 256), (2048, 512), (5120, 1536)])
def test_experts_defaults_are_tested(hb, gpu, hidden, inter):
    """One form a tile size and product, whatever the sizes: those of the GPU tests."""
    for bm, gate_up in [(32, True), (64, True), (128, True), (32, False), (64, False), (128, False)]:
        k, n, out, rows = (hidden, 2 * inter, hb.Out.Swiglu, hb.Rows.Gather) if gate_up else (inter, hidden, hb.Out.Bf16, hb.Rows.Scatter)
        tags = {re.search("_t.*?(?=_gather|_scatter)", gpu.kernel_name(gpu.pipeline(hb.experts_f8(a, b, out, rows, 2, 5, 100, bm)))).group()
                for a, b in ((k, n), (400, 512))}
        assert len(tags) == 1, tags


def test_sums(hb, gpu):
    """f32 sums are a kernel of their own for outputs of two bytes and the SwiGLU, and none for f32's; other
    values of the part are refused."""
    for out in hb.Out:
        names = {gpu.kernel_name(gpu.pipeline(hb.gemm_f8(2560, 512, out, rows=64, f32_sums=f))) for f in (False, True)}
        assert len(names) == (1 if out == hb.Out.F32 else 2), names
    for bm, n in ((16, 1), (64, 2)):
        made = [hb.experts_f8(256, 512, hb.Out.Swiglu, hb.Rows.Gather, 2, 8, 64, bm, f32_sums=f) for f in (False, True)]
        assert len({gpu.kernel_name(gpu.pipeline(d)) for d in made}) == n
    with pytest.raises(hb.HerbertError, match="sums"):
        gpu.pipeline(hb.gemm_f8(2560, 512, hb.Out.Bf16).replace(form=2))


def test_matvec_defaults_are_tested(hb, gpu):
    """The same of the matvec's forms, dense and over experts; a form of more than 8 x rows is tested
    there with 10 and 16."""
    import test_gpu_f8_mv_forms as forms

    taken = {False: set(), True: set()}
    rng = random.Random(7)

    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    for _ in range(6000):
        k, m, experts = 16 * size(1, 1088), size(1, 16), rng.random() < 0.3
        if experts:
            gate_up = rng.random() < 0.5
            d = hb.experts_f8(k, 256 * size(1, 40), hb.Out.Swiglu if gate_up else hb.Out.Bf16, hb.Rows.Gather if gate_up else hb.Rows.Scatter,
                              rng.choice([1, 2, 4, 8]), rng.choice([8, 64, 256]), m, 16)
        else:
            out = rng.choice(list(hb.Out))
            d = hb.matvec_f8(k, 256 * size(1, 136) if out == hb.Out.Swiglu else size(16, 151936), out, mv_m=m)
        f = tuple(int(v) for v in re.search(r"_r(\d+)_k(\d+)_w(\d+)_u(\d+)_m", gpu.kernel_name(gpu.pipeline(d))).groups())
        assert experts or (f in forms.FORMS and (f != forms.FORMS[1] or m <= 8)), (f, m)
        taken[experts].add(f)
    assert taken[False] == set(forms.FORMS)
    # The experts' by their cases there: few pairs and many, long K and short.
    made = set()
    for t, k, n in [(40, 1040, 512), (2, 1040, 512), (2, 272, 256), (2, 144, 256), (2, 128, 256), (60, 272, 512)]:
        for out, rows in ((hb.Out.Swiglu, hb.Rows.Gather), (hb.Out.Bf16, hb.Rows.Scatter)):
            name = gpu.kernel_name(gpu.pipeline(hb.experts_f8(k, n, out, rows, 2, 3, t, 16)))
            made.add(tuple(int(v) for v in re.search(r"_r(\d+)_k(\d+)_w(\d+)_u(\d+)_m", name).groups()))
    assert taken[True] <= made, taken[True] - made
