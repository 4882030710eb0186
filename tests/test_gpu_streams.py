"""The context on a caller's stream (hb_set_stream): its launches and graph
replays stand in one order with the caller's own work there, with nothing
waited for in between."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

import herbert_hip as hb
import q4_ref as q4

pytestmark = pytest.mark.gpu

K, N, M, GROUP = 1024, 512, 3, 64
D2D = 3  # hipMemcpyDeviceToDevice


class Hip:
    """A few calls of the HIP runtime that the library itself is bound to."""

    def __init__(self):
        self.lib = ctypes.CDLL(sorted(hb._hip_runtimes())[0])

    def __call__(self, name, *args):
        rc = getattr(self.lib, name)(*args)
        assert rc == 0, (name, rc)

    def stream(self):
        s = ctypes.c_void_p()
        self("hipStreamCreateWithFlags", ctypes.byref(s), 1)
        return s


def pointer(gpu, buf):
    p = ctypes.c_void_p()
    hb.check(hb.lib.hb_buffer_ptr(gpu.h, buf, ctypes.byref(p)))
    return p


@pytest.mark.parametrize("null", [False, True])
@pytest.mark.parametrize("graph", [False, True])
def test_in_order_with_the_callers_work(gpu, null, graph):
    """Per turn, on one stream and with no wait: a long copy, the turn's x into
    the bound buffer, the matvec, y into the turn's place.  Each y belongs to
    its turn's x."""
    if len(hb._hip_runtimes()) > 1:
        pytest.skip("two HIP runtimes in this process")
    hip, turns, big = Hip(), 12, 256 << 20
    rng = np.random.default_rng(21)
    codes, scales = q4.exact_codes(rng, N, K, GROUP)
    xs = hb.f32_to_bf16(rng.integers(-4, 5, (turns, M, K)).astype(np.float32))
    w = q4.pack(gpu, codes, scales, K, N, GROUP)
    kern = gpu.pipeline(hb.matvec_q4(K, N, hb.Out.F32, GROUP, M))
    src, x, y = gpu.alloc_with(xs), gpu.alloc_with(np.zeros((M, K), np.uint16)), gpu.alloc_with(np.zeros((M, N), np.float32))
    out, a, b = gpu.alloc(turns * M * N * 4), gpu.alloc(big), gpu.alloc(big)
    ranges = [hb.r(w), hb.r(x), hb.r(y)]
    run = gpu.graph([hb.Op(kern, ranges, M)]) if graph else None
    gpu.sync()
    stream = ctypes.c_void_p() if null else hip.stream()
    p = {name: pointer(gpu, buf).value for name, buf in (("src", src), ("x", x), ("y", y), ("out", out), ("a", a), ("b", b))}

    def copy(to, at, frm, off, size):
        hip("hipMemcpyAsync", ctypes.c_void_p(p[to] + at), ctypes.c_void_p(p[frm] + off), ctypes.c_size_t(size), D2D, stream)

    try:
        gpu.set_stream(stream.value or 0)
        for t in range(turns):
            copy("b", 0, "a", 0, big)
            copy("x", 0, "src", t * M * K * 2, M * K * 2)
            run.launch() if graph else gpu.launch(kern, ranges, M)
            copy("out", t * M * N * 4, "y", 0, M * N * 4)
        gpu.set_stream()  # waits for the turns
        got = gpu.download(out, np.float32, turns * M * N).reshape(turns, M, N)
    finally:
        gpu.set_stream()
        if run:
            run.free()
        if not null:
            hip("hipStreamDestroy", stream)
        for buf in (w, src, x, y, out, a, b):
            gpu.free(buf)
    want = hb.bf16_to_f32(xs).astype(np.float64) @ q4.values(codes, scales, GROUP).T
    assert np.array_equal(got.astype(np.float64), want)


def test_split_gemm_and_timing_on_a_callers_stream(gpu):
    """What uses the workspace and the events gives the same there."""
    if len(hb._hip_runtimes()) > 1:
        pytest.skip("two HIP runtimes in this process")
    hip, (m, k, n) = Hip(), (64, 2048, 256)
    x, w = hb.normal_bf16(1, 1.0, (m, k)), hb.normal_bf16(2, 0.02, (n, k))
    bufs = [gpu.alloc_with(v) for v in (np.array([0, 0, 0, m], np.uint32), w, x, np.zeros((m, n), np.uint16))]
    st, wb, xb, yb = bufs
    kern = gpu.pipeline(hb.gemm_mma(k, n, hb.Out.Bf16, bm=64, bn=64, bk=64, wm=2, wn=2, mfma=16, dbuf=1, lds_dma=1, order=1, ksplit=4))
    op = [hb.r(st), hb.r(wb), hb.r(xb), hb.r(yb), hb.r(st), hb.r(st)]
    stream = hip.stream()
    try:
        gpu.launch(kern, op, m)
        want = gpu.download(yb, np.uint16, m * n)
        gpu.zero(yb)
        gpu.set_stream(stream.value)
        gpu.launch(kern, op, m)
        assert np.array_equal(gpu.download(yb, np.uint16, m * n), want)
        gpu.zero(yb)
        assert gpu.time_ops([hb.Op(kern, op, m)], 3) > 0
        assert np.array_equal(gpu.download(yb, np.uint16, m * n), want)
    finally:
        gpu.set_stream()
        hip("hipStreamDestroy", stream)
        for b in bufs:
            gpu.free(b)


TORCH = r"""
import ctypes, sys
import torch
sys.path[:0] = sys.argv[1:3]
import herbert_hip as hb, q4_ref as q4
import numpy as np

K, N, M, GROUP = 1024, 512, 3, 64
g = hb.Gpu(0)


class View:
    def __init__(self, buf, shape, typestr):
        p = ctypes.c_void_p()
        hb.check(hb.lib.hb_buffer_ptr(g.h, buf, ctypes.byref(p)))
        self.__cuda_array_interface__ = {"shape": shape, "typestr": typestr, "data": (p.value, False), "version": 2}


def tensor(buf, shape, typestr):
    return torch.as_tensor(View(buf, shape, typestr), device="cuda")


rng = np.random.default_rng(5)
codes, scales = q4.exact_codes(rng, N, K, GROUP)
w = q4.pack(g, codes, scales, K, N, GROUP)
xs = torch.from_numpy(rng.integers(-4, 5, (8, M, K)).astype(np.float32)).to("cuda", torch.bfloat16)
want = xs.double().cpu().numpy() @ q4.values(codes, scales, GROUP).T
xb, yb = g.alloc_with(np.zeros((M, K), np.uint16)), g.alloc_with(np.zeros((M, N), np.float32))
x, y = tensor(xb, (M, K), "<i2").view(torch.bfloat16), tensor(yb, (M, N), "<f4")
kern = g.pipeline(hb.matvec_q4(K, N, hb.Out.F32, GROUP, M))
ranges = [hb.r(w), hb.r(xb), hb.r(yb)]
slow = torch.randn(4096, 4096, device="cuda")


def turns(what):
    outs = []
    for t in range(8):
        z = slow @ slow
        x.copy_(xs[t])
        g.launch(kern, ranges, M)
        outs.append(y.clone())
    torch.cuda.synchronize()
    got = torch.stack(outs).double().cpu().numpy()
    assert np.array_equal(got, want), what
    print("ok", what, flush=True)


torch.cuda.synchronize()
g.set_stream(torch.cuda.current_stream().cuda_stream)
turns("torch's default stream")
side = torch.cuda.Stream()
torch.cuda.synchronize()
g.set_stream(side.cuda_stream)
with torch.cuda.stream(side):
    turns("a side stream")
    # Captured there with torch's own work, and replayed with eager work between.
    graph = torch.cuda.CUDAGraph()
    at = xs[0].clone()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        x.copy_(at)
        g.launch(kern, ranges, M)
        z = y * 2
    for turn in range(3):
        for t in (3, 0, 7, 5):
            at.copy_(xs[t])
            graph.replay()
            got = z.clone()
            x.copy_(xs[1])
            g.launch(kern, ranges, M)
            eager = y.clone()
            torch.cuda.synchronize()
            assert np.array_equal(got.double().cpu().numpy(), 2 * want[t]), (turn, t)
            assert np.array_equal(eager.double().cpu().numpy(), want[1]), (turn, t)
print("ok capture", flush=True)
del graph
torch.cuda.synchronize()
g.set_stream()
g.launch(kern, ranges, M)
assert np.array_equal(g.download(yb, np.float32, M * N).reshape(M, N), want[1])
g.close()
print("ok all", flush=True)
"""


def test_tensors_over_the_buffers():
    """In a process that imports torch first: torch's default stream, a side
    stream, and a capture by torch that holds the library's launches."""
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-u", "-c", TORCH, os.path.dirname(os.path.dirname(os.path.abspath(hb.__file__))), here],
                       capture_output=True, text=True, timeout=110)
    print(r.stdout, r.stderr, flush=True)
    assert r.returncode == 0 and r.stdout.splitlines()[-1] == "ok all", r.stderr
